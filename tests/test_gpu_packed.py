"""Attention over sequences that lie one behind the other, and its gradients, against float64 (window_reference, a sequence at a time)."""
import threading

import pytest
import torch

from mojodiffusion_amd import attention_packed as P
from mojodiffusion_amd import attention_window as W
from mojodiffusion_amd.attention_sage import Error
from window_reference import backward, check_backward, check_forward, forward

BF, FP = torch.bfloat16, torch.float16
NAN = float("nan")

CASES = [
    # query rows by sequence, key rows by sequence (None: the same), Hq, Hk, D, type, causal, rows behind the last sequence
    ([1], None, 1, 1, 64, BF, True, 0),
    ([5, 1, 33, 64], None, 4, 2, 128, BF, True, 3),
    ([100, 0, 7, 257], None, 3, 1, 64, FP, True, 0),
    ([31, 32, 33], None, 2, 2, 256, FP, False, 40),
    ([0, 0, 129, 0], None, 12, 4, 128, FP, False, 1),
    ([n * 7 % 23 for n in range(130)], None, 2, 1, 64, BF, True, 5),
    ([3, 40, 1], [50, 40, 300], 6, 3, 64, BF, True, 2),
    ([40, 5, 9, 2], [3, 0, 9, 1], 5, 1, 128, BF, True, 7),
    ([40, 5, 9], [3, 0, 70], 8, 8, 64, FP, False, 0),
    ([200, 17, 300], [210, 500, 300], 16, 2, 256, BF, True, 0),
    # workgroups of 128 rows
    ([300, 1, 513, 129, 90], None, 12, 12, 128, BF, True, 70),
    ([640, 90, 333], None, 24, 8, 64, BF, True, 0),
    ([410, 77, 333, 200], None, 18, 18, 256, FP, False, 9),
    ([200, 333, 128], [100, 400, 129], 40, 10, 64, FP, True, 1),
    ([500, 400, 300], None, 30, 30, 64, BF, False, 0),
    ([650], None, 7, 7, 64, FP, True, 0),
]


def offsets(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32)


def tensors(nq, nk, Hq, Hk, D, dtype, tail, seed):
    g = torch.Generator().manual_seed(seed)
    q, k, v, d = (torch.randn((sum(n) + tail, h, D), generator=g).to(dtype) for n, h in ((nq, Hq), (nk, Hk), (nk, Hk), (nq, Hq)))
    k += 0.5 * torch.randn((1, Hk, D), generator=g).to(dtype)
    return q, k, v, d


def per_sequence(nq, nk, q, k, v, causal, scale):
    """(rows of q, rows of k, reference) of every sequence with queries and keys."""
    a = b = 0
    for n, m in zip(nq, nk):
        if n and m:
            yield slice(a, a + n), slice(b, b + m), forward(q[None, a:a + n], k[None, b:b + m], v[None, b:b + m], scale, -1, 0 if causal else -1, 0, [m], [m - n])
        a, b = a + n, b + m


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nk,Hq,Hk,D,dtype,causal,tail", CASES)
def test_packed(nq, nk, Hq, Hk, D, dtype, causal, tail):
    own = nk is not None
    nk = nk or nq
    q, k, v, d = tensors(nq, nk, Hq, Hk, D, dtype, tail, sum(nq) + D)
    scale = D ** -0.5
    real_q, real_k = torch.zeros(q.shape[0], dtype=torch.bool), torch.zeros(k.shape[0], dtype=torch.bool)
    refs = list(per_sequence(nq, nk, q, k, v, causal, scale))
    for rq, rk, ref in refs:
        real_q[rq], real_k[rk] = (ref[2][0].sum(2) > 0).any(0), (ref[2][0].sum(1) > 0).any(0)
    # what sees nothing, is seen by nothing or belongs to no sequence may hold anything
    q[~real_q], d[~real_q], k[~real_k], v[~real_k] = NAN, NAN, NAN, NAN
    cu, cu_k = offsets(nq).cuda(), offsets(nk).cuda() if own else None
    args = (q.cuda(), k.cuda(), v.cuda(), cu, scale, causal, cu_k)
    o = P.sdpa_packed(*args)
    fwd = P.sdpa_packed_train_fwd(*args)
    assert torch.equal(fwd.o, o) and (o[~real_q] == 0).all() and torch.isneginf(fwd.stats[:, ~real_q]).all()
    for rq, rk, ref in refs:
        check_forward(o[None, rq], fwd.stats[None, :, rq], ref, dtype)
    # the Python path: int64 offsets, rows of a wider tensor
    wide = torch.zeros((q.shape[0], Hq + 1, D), dtype=dtype).cuda()
    wide[:, 1:] = args[0]
    assert torch.equal(P.sdpa_packed(wide[:, 1:], *args[1:3], cu.long(), scale, causal, None if cu_k is None else cu_k.long()), o)
    if D == 256:
        with pytest.raises(Error, match="Dh=256"):
            P.sdpa_packed_backward(fwd, d.cuda())
        return
    got = P.sdpa_packed_backward(fwd, d.cuda())
    assert (got.d_q[~real_q] == 0).all() and (got.d_k[~real_k] == 0).all() and (got.d_v[~real_k] == 0).all()
    for rq, rk, ref in refs:
        some = real_k[rk].nonzero().view(-1)
        clean = [torch.where(torch.isnan(t), torch.zeros_like(t), t) for t in (q[None, rq], k[None, rk], v[None, rk], d[None, rq])]
        check_backward([t[None, r] for t, r in ((got.d_q, rq), (got.d_k, rk), (got.d_v, rk))], backward(*clean, scale, ref, Hq // Hk))
        assert some.numel()
    again = P.sdpa_packed_backward(P.SdpaPackedFwd(**{**fwd.__dict__, "cu_seqlens": cu.long(), "cu_seqlens_k": None if cu_k is None else cu_k.long()}), d.cuda())
    for x, y in zip((again.d_q, again.d_k, again.d_v), (got.d_q, got.d_k, got.d_v)):
        assert torch.equal(x, y)


FORMS = [
    # workgroups of 128 rows with a wave or two to 32 rows, all head dims, rows that see nothing among them
    ([300, 1, 513, 129, 90], None, 24, 8, 128, BF, True, 70),
    ([300, 1, 513, 129, 90], None, 60, 12, 128, FP, True, 5),
    ([333, 70, 500], [333, 31, 900], 24, 24, 128, FP, False, 0),
    ([200, 333, 128], [100, 400, 129], 32, 32, 128, BF, True, 1),
    ([600, 1, 401], None, 18, 6, 256, BF, True, 3),
    ([600, 1, 401], [40, 33, 500], 36, 36, 256, FP, True, 3),
    ([100, 333, 64, 31, 600], None, 22, 11, 64, BF, False, 1),
    ([1100], [1200], 20, 4, 64, FP, True, 0),
    ([1111], None, 24, 24, 64, BF, True, 9),
    ([95, 1030], [1500, 2100], 10, 10, 128, BF, True, 0),
]
LONG_WALKS = [
    # few rows that walk many keys: gradients in parts; queries before the first key among them
    ([900], [700], 6, 2, 64, BF, True, 3),
    ([900], [700], 4, 4, 128, FP, True, 0),
    ([600], [2000], 8, 2, 128, BF, False, 2),
    ([1, 1], [1800, 600], 4, 4, 64, FP, True, 0),
    ([700, 0, 300], [900, 1400, 40], 3, 1, 128, BF, True, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nk,Hq,Hk,D,dtype,causal,tail", FORMS)
def test_packed_in_larger_grids(nq, nk, Hq, Hk, D, dtype, causal, tail):
    test_packed(nq, nk, Hq, Hk, D, dtype, causal, tail)


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nk,Hq,Hk,D,dtype,causal,tail", LONG_WALKS)
def test_packed_long_walks(nq, nk, Hq, Hk, D, dtype, causal, tail):
    test_packed(nq, nk, Hq, Hk, D, dtype, causal, tail)


@pytest.mark.gpu
def test_more_sequences_than_lanes_in_a_large_grid():
    lens = [(b * 37) % 61 for b in range(70)] + [300, 0, 5]
    T = sum(lens)
    q, k, v, _ = (t.cuda() for t in tensors(lens, lens, 16, 16, 64, FP, 11, 7))
    assert T * 16 // 128 > 256
    o = P.sdpa_packed(q, k, v, offsets(lens).cuda(), 0.125)
    assert (o[T:] == 0).all()
    at = 0
    for n in lens:
        r, at = slice(at, at + n), at + n
        if n:
            check_forward(o[None, r], None, forward(q[None, r], k[None, r], v[None, r], 0.125, -1, 0, 0, [n], [0]), FP)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [64, 65, 90])
@pytest.mark.parametrize("causal", [True, False])
def test_many_sequences(B, causal):
    """As many as one lane each takes, and more, in workgroups of 128 rows: every sequence as it is alone among few."""
    lens = [(b * 37) % 61 for b in range(B - 1)] + [200]
    T = sum(lens)
    q, k, v, d = (t.cuda() for t in tensors(lens, lens, 12, 12, 64, BF, 6, B))
    f = P.sdpa_packed_train_fwd(q, k, v, offsets(lens).cuda(), 0.125, causal)
    g = P.sdpa_packed_backward(f, d)
    for t in (f.o, g.d_q, g.d_k, g.d_v):
        assert (t[T:] == 0).all()
    assert torch.isneginf(f.stats[:, T:]).all()
    at = 0
    for b, n in enumerate(lens):
        r, at = slice(at, at + n), at + n
        if not n or (b % 7 and n != 200):
            continue
        ref = forward(q[None, r], k[None, r], v[None, r], 0.125, -1, 0 if causal else -1, 0, [n], [0])
        check_forward(f.o[None, r], f.stats[None, :, r], ref, BF)
        check_backward([t[None, r] for t in (g.d_q, g.d_k, g.d_v)], backward(*(t[None, r] for t in (q, k, v, d)), 0.125, ref, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("D,dtype,causal", [(64, BF, True), (128, FP, True), (128, BF, False)])
def test_gradients_against_differences(D, dtype, causal):
    """The slope of sum(O d) along a direction, from differences of the float64 forward, and the recorded node's gradients: no further apart than the bounds of
    the gradients allow (and 1e-6 of the slope's size, for the differences' own error: third derivatives times the step's square, 1e-4 squared)."""
    nq, Hq, Hk, scale = [40, 9, 70], 4, 2, D ** -0.5
    q, k, v, d = tensors(nq, nq, Hq, Hk, D, dtype, 0, 3)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    P.record_sdpa_packed(*leaves, offsets(nq).cuda(), scale, causal).backward(d.cuda())
    g = torch.Generator().manual_seed(4)
    for i, x in enumerate((q, k, v)):
        u = torch.randn(x.shape, generator=g).double()

        def value(step):
            moved = [t.double() + (step * u if t is x else 0) for t in (q, k, v)]
            return sum(float((ref[0][0] * d[rq].double()).sum()) for rq, _, ref in per_sequence(nq, nq, *moved, causal, scale))

        slope = (value(1e-4) - value(-1e-4)) / 2e-4
        got = float((leaves[i].grad.cpu().double() * u).sum())
        bound, size = 0.0, 0.0
        for rq, rk, ref in per_sequence(nq, nq, q, k, v, causal, scale):
            want, limit = backward(q[None, rq], k[None, rk], v[None, rk], d[None, rq], scale, ref, Hq // Hk)[i]
            bound, size = bound + float((limit[0] * u[rq].abs()).sum()), size + float((want[0].abs() * u[rq].abs()).sum())
        assert abs(got - slope) <= bound + 1e-6 * size, (i, got, slope, bound)


@pytest.mark.gpu
def test_one_sequence_is_causal_windowed_attention():
    """One sequence through both operators: the same values to the bounds' rounding, and both kinds of workgroups the same as themselves when a batch has more of them."""
    q, k, v, d = (t.cuda() for t in tensors([700], [700], 12, 4, 128, BF, 0, 8))
    one = P.sdpa_packed(q, k, v, offsets([700]).cuda(), 0.1)
    other = W.sdpa_window(q[None], k[None], v[None], 0.1, -1, 0)[0]
    assert (one.float() - other.float()).abs().max() <= 2.0 ** -7 * one.float().abs().max()
    many = P.sdpa_packed(*(t.repeat(6, 1, 1) for t in (q, k, v)), offsets([700] * 6).cuda(), 0.1).view(6, 700, 12, 128)
    for x in many:
        assert torch.equal(x, many[0])
    f = P.sdpa_packed_train_fwd(*(t.repeat(6, 1, 1) for t in (q, k, v)), offsets([700] * 6).cuda(), 0.1)
    g = P.sdpa_packed_backward(f, d.repeat(6, 1, 1))
    for t in (g.d_q, g.d_k, g.d_v):
        for x in t.view(6, 700, -1, 128):
            assert torch.equal(x, t[:700])


@pytest.mark.gpu
def test_offsets_beyond_the_rows():
    """Offsets past the last row end there; the first one counts as 0."""
    q, k, v, d = (t.cuda() for t in tensors([60], [60], 4, 2, 64, BF, 0, 1))
    want = P.sdpa_packed_train_fwd(q, k, v, torch.tensor([0, 25, 60]).cuda(), 0.125)
    got = P.sdpa_packed_train_fwd(q, k, v, torch.tensor([7, 25, 2 ** 31 - 1], dtype=torch.int32).cuda(), 0.125)
    assert torch.equal(got.o, want.o) and torch.equal(got.stats, want.stats)
    a, b = (P.sdpa_packed_backward(f, d) for f in (want, got))
    assert torch.equal(a.d_q, b.d_q) and torch.equal(a.d_k, b.d_k) and torch.equal(a.d_v, b.d_v)


@pytest.mark.gpu
def test_rows_beyond_32_bit_offsets():
    """300000 rows, 8192 elements apart: the last sequence lies more than 2^31 elements in."""
    wide = torch.zeros((300000, 64, 128), dtype=BF, device="cuda")
    q, k, v, _ = tensors([50], [50], 1, 1, 128, BF, 0, 2)
    n = 299950
    for i, t in enumerate((q, k, v)):
        wide[n:, i:i + 1] = t.cuda()
    o = P.sdpa_packed(wide[:, 0:1], wide[:, 1:2], wide[:, 2:3], torch.tensor([0, 100, n - 300, n, 300000], dtype=torch.int32).cuda(), 0.1)
    check_forward(o[None, n:], None, forward(q[None], k[None], v[None], 0.1, -1, 0, 0, [50], [0]), BF)
    assert (o[:n] == 0).all()


@pytest.mark.gpu
def test_a_captured_training_step():
    """Replayed with other values and other lengths between, against the eager step."""
    Hq, Hk, D, T = 6, 2, 64, 900
    lens = [[300, 1, 599], [899, 0, 0], [100, 400, 333]]
    sets = [tensors([T], [T], Hq, Hk, D, BF, 0, s) for s in range(3)]

    def step(q, k, v, d, cu):
        f = P.sdpa_packed_train_fwd(q, k, v, cu, 0.125)
        g = P.sdpa_packed_backward(f, d)
        return f.o, f.stats, g.d_q, g.d_k, g.d_v

    eager = [[t.clone() for t in step(*(t.cuda() for t in s), offsets(n).cuda())] for s, n in zip(sets, lens)]
    place = [t.cuda() for t in sets[0]]
    cu = offsets(lens[0]).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*place, cu)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*place, cu)
    for i in (0, 1, 2, 1):
        for t, x in zip(place, sets[i]):
            t.copy_(x)
        cu.copy_(offsets(lens[i]))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, eager[i]):
            assert torch.equal(x, y), i
        step(*(t.cuda() for t in sets[0]), offsets(lens[2]).cuda())


# workgroups of 128 rows, with two waves to 32 rows, and of 32
BY_FORM = [(700, 56), (500, 40), (300, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,H", BY_FORM)
@pytest.mark.parametrize("D,dtype", [(64, FP), (128, BF), (256, BF)])
@pytest.mark.parametrize("causal", [True, False])
def test_scores_that_rise_and_fall(T, H, D, dtype, causal):
    """Every tile's largest score far above the one before's, in half of the heads far below: the running reference is raised on every tile, or on the first alone."""
    q, k, v, _ = tensors([T], [T], H, H, D, dtype, 0, T + D)
    q[:] = q[:1].abs() + 0.25                # (all queries one direction, that of the keys)
    size = torch.linspace(0.05, 6.0, T).view(-1, 1)
    k = (k * 0.05).double()
    k[:, : H // 2] += (size * 1.0).unsqueeze(2)
    k[:, H // 2:] += (size.flip(0) * 1.0).unsqueeze(2)
    k = k.to(dtype)
    scale = 4.0 / D
    f = P.sdpa_packed_train_fwd(q.cuda(), k.cuda(), v.cuda(), offsets([T]).cuda(), scale, causal)
    ref = forward(q[None], k[None], v[None], scale, -1, 0 if causal else -1, 0, [T], [0])
    assert float(ref[1].max()) > 15
    check_forward(f.o[None], f.stats[None], ref, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("T,H", BY_FORM)
@pytest.mark.parametrize("D", [64, 128])
def test_queries_that_are_not_finite(T, H, D):
    """A NaN or an infinity in a query: NaN in its own row, and every other row within its bounds."""
    q, k, v, _ = tensors([T - 40, 40], [T - 40, 40], H, H, D, BF, 0, 9)
    cu = offsets([T - 40, 40]).cuda()
    refs = list(per_sequence([T - 40, 40], [T - 40, 40], q, k, v, True, 0.1))
    bad = [(3, 0), (100, 1), (T - 1, H - 1), (T - 50, 2)]
    for value in (NAN, float("inf"), -float("inf")):
        x = q.clone()
        for i, h in bad:
            x[i, h, 7] = value
        o = P.sdpa_packed(x.cuda(), k.cuda(), v.cuda(), cu, 0.1)
        clean = P.sdpa_packed(q.cuda(), k.cuda(), v.cuda(), cu, 0.1)
        for i, h in bad:
            assert torch.isnan(o[i, h]).all()
            o[i, h] = clean[i, h]
        for rq, _, ref in refs:
            check_forward(o[None, rq], None, ref, BF)


@pytest.mark.gpu
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, FP)])
def test_other_orders_in_memory(D, dtype):
    """Heads first, rows far apart, an upstream gradient that is one row repeated, rows that are not aligned (copied): the bits of dense tensors."""
    lens = [70, 130, 9]
    T, Hq, Hk = sum(lens), 6, 3
    q, k, v, d = (t.cuda() for t in tensors(lens, lens, Hq, Hk, D, dtype, 0, D))
    d = d[:1].expand(T, Hq, D)
    cu = offsets(lens).cuda()

    def step(q, k, v, d):
        f = P.sdpa_packed_train_fwd(q, k, v, cu, 0.1)
        g = P.sdpa_packed_backward(f, d)
        return f.o, f.stats, g.d_q, g.d_k, g.d_v

    want = step(q, k, v, d.contiguous())
    heads_first = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)

    def apart(t):
        w = torch.full((2 * t.shape[0], t.shape[1] + 2, 2 * D), NAN, dtype=dtype, device="cuda")
        w[1::2, 1:-1, D:] = t
        return w[1::2, 1:-1, D:]

    def unaligned(t):
        w = torch.zeros(t.numel() + 1, dtype=dtype, device="cuda")[1:].view(t.shape)
        w.copy_(t)
        return w

    for order in (heads_first, apart, unaligned):
        for x, y in zip(step(order(q), order(k), order(v), d), want):
            assert torch.equal(x, y)
        for x, y in zip(step(q, order(k), order(v), order(d.contiguous())), want):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_a_captured_recorded_step():
    """The recorded node in a captured forward and backward (the warm-up's graph and gradients are gone by then), replayed with other values between."""
    Hq, Hk, D, T = 6, 2, 128, 260
    lens = [[100, 160], [1, 259]]
    sets = [tensors([T], [T], Hq, Hk, D, FP, 0, s) for s in range(2)]

    def step(q, k, v, d, cu):
        o = P.record_sdpa_packed(q, k, v, cu, 0.1)
        return (o.detach(), *torch.autograd.grad(o, (q, k, v), d))

    eager = []
    for s, n in zip(sets, lens):
        q, k, v, d = (t.cuda() for t in s)
        eager.append([t.clone() for t in step(*(t.requires_grad_() for t in (q, k, v)), d, offsets(n).cuda())])
        del q, k, v, d
    place = [t.cuda() for t in sets[0]]
    leaves = [t.requires_grad_() for t in place[:3]]
    cu = offsets(lens[0]).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*leaves, place[3], cu)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*leaves, place[3], cu)
    for i in (0, 1, 1, 0):
        with torch.no_grad():
            for t, x in zip(place, sets[i]):
                t.copy_(x)
        cu.copy_(offsets(lens[i]))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, eager[i]):
            assert torch.equal(x, y), i


@pytest.mark.gpu
def test_two_threads_on_streams_of_their_own():
    cu = offsets([200, 100]).cuda()
    sets = [[t.cuda() for t in tensors([300], [300], 4, 2, 128, BF, 0, s)] for s in range(2)]
    step = lambda q, k, v, d: P.sdpa_packed_backward(P.sdpa_packed_train_fwd(q, k, v, cu, 0.1), d)
    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                g = step(*sets[i])
                if not all(torch.equal(a, b) for a, b in zip((g.d_q, g.d_k, g.d_v), (want[i].d_q, want[i].d_k, want[i].d_v))):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


@pytest.mark.gpu
def test_a_trained_projection():
    """The recorded node between torch's own: a joint projection, whose parts go in as they are, and an upstream gradient that is not dense."""
    g = torch.Generator().manual_seed(6)
    x, w = (torch.randn(s, generator=g).to(BF).cuda() for s in ((90, 64), (64, 6 * 64)))
    w = (w * 0.125).requires_grad_()
    cu = offsets([30, 60]).cuda()
    qkv = (x @ w).view(90, 6, 64)
    o = P.record_sdpa_packed(qkv[:, :4], qkv[:, 4:5], qkv[:, 5:], cu, 0.125)
    o.transpose(0, 1).float().square().sum().backward()
    d_o = 2 * o.detach().float()
    f = P.sdpa_packed_train_fwd(*(t.detach().contiguous() for t in (qkv[:, :4], qkv[:, 4:5], qkv[:, 5:])), cu, 0.125)
    s = P.sdpa_packed_backward(f, d_o.to(BF))
    want = x.float().T @ torch.cat((s.d_q, s.d_k, s.d_v), 1).view(90, -1).float()
    # (torch's product: bf16 operands, fp32 sums, one rounding to bf16, 2^-8, with room for a sum of 90 terms)
    assert ((w.grad.float() - want).abs() <= 2.0 ** -8 * want.abs() + 90 * 2.0 ** -23 * (x.float().abs().T @ torch.cat((s.d_q, s.d_k, s.d_v), 1).view(90, -1).float().abs())).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,H", [(64, 2), (1024, 24), (1024, 56)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_fp16_weights_below_the_normal_range(T, H, D):
    """The first keys of four tiles far above the others, and with values of zero: what comes out is the sum of 8000 weights of 2^-25.5 of the largest each, which the statistics count as well.
    Such a weight is off by 2^-32 of the largest at the most.  (All rows alike: one of them is the reference.)  In all three forms."""
    n = 8200
    g = torch.Generator().manual_seed(D)
    k, v = torch.zeros((n, 1, D)), 16 * (1 + torch.rand((n, 1, D), generator=g))
    k[0:128:32, 0, 0], v[0:128:32] = 16.0, 0.0
    q = torch.zeros((1, 1, D))
    q[..., 0] = 25.5 * 0.6931 / 16 / 0.125
    q, k, v = (t.to(FP) for t in (q, k, v))
    O, L, W, A, F, E = forward(q[None], k[None], v[None], 0.125, -1, -1, 0, [n], [0])
    assert W[..., 1].max() < 2.0 ** -25.2 * W[..., 0].min() and O.min() > 2.0 ** -12
    f = P.sdpa_packed_train_fwd(q.expand(T, H, D).contiguous().cuda(), *(t.expand(n, H, D).contiguous().cuda() for t in (k, v)), offsets([T]).cuda(), 0.125, False, offsets([n]).cuda())
    bound = 2.0 ** -11 * O.abs() + A * (1.01 * 2.0 ** -11 + n * 2.0 ** -24 + 2.1 * E.transpose(1, 2).unsqueeze(-1)) + F * 2.0 ** -32 + 2.0 ** -25
    err = (f.o.cpu().double() - O[0]).abs()
    assert (err <= bound[0]).all(), float((err / bound[0]).max())
    assert ((f.stats.cpu().double() - L[0, 0, 0]).abs() <= E[0, 0, 0] + n * 2.0 ** -24).all()


PADDED = [
    # a batch of fixed B whose last, first or other sequences are empty: gradients in parts (keys' pairs and rows' key tiles), two waves to 32 rows
    ([3000, 0, 0, 0, 0], None, 1, 1, 64, BF, True, 0),
    ([0, 2200, 0, 700, 0], None, 4, 2, 128, FP, False, 3),
    ([0, 0, 1500], None, 12, 12, 128, BF, True, 0),
    ([0, 1500, 0], [0, 1700, 0], 12, 12, 64, FP, False, 2),
    ([0] * 63 + [900], None, 2, 1, 64, BF, True, 1),
    ([900] + [0] * 80, None, 3, 3, 128, FP, True, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nk,Hq,Hk,D,dtype,causal,tail", PADDED)
def test_packed_with_empty_sequences(nq, nk, Hq, Hk, D, dtype, causal, tail):
    test_packed(nq, nk, Hq, Hk, D, dtype, causal, tail)
