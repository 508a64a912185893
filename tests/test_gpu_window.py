"""Attention over a sliding window: sdpa_window, sdpa_window_train_fwd and sdpa_window_decode against the definition in float64 (bounds:
window_reference.forward)."""
import pytest
import torch

from mojodiffusion_amd import attention_window as W
from mojodiffusion_amd.attention_sage import Error
from window_reference import backward, check_backward, check_forward, forward

BF, FP = torch.bfloat16, torch.float16


def tensors(B, Sq, Skv, Hq, Hk, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(s, generator=g)
    k = make(B, Skv, Hk, D) + 0.5 * make(B, 1, Hk, D)
    return make(B, Sq, Hq, D).to(dtype), k.to(dtype), make(B, Skv, Hk, D).to(dtype)


# Few rows (keys split over waves and workgroups) and many (tiles shared by a workgroup's waves); one query, one key; windows of one key, of whole
# tiles and one more or less; sinks inside, at and behind a tile's end, more than there are keys; right edges; no left edge, no edge at all;
# sequences of length 0, 1 and others; queries before the first key and behind the last; odd groups of heads.
CASES = [
    # B, Sq, Skv, Hq, Hk, D, type, left, right, sinks, lens, first
    (1, 1, 1, 1, 1, 64, BF, 0, 0, 0, None, 0),
    (2, 5, 7, 2, 1, 128, FP, 1, 0, 1, None, 2),
    (1, 33, 33, 3, 3, 64, BF, 7, 0, 4, None, 0),
    (1, 100, 100, 2, 2, 256, FP, 16, 16, 0, None, 0),
    (3, 65, 200, 4, 2, 128, BF, 63, 0, 64, [200, 0, 1], 120),
    (2, 64, 64, 5, 1, 64, BF, -1, 0, 0, None, 0),
    (2, 31, 129, 2, 2, 128, BF, -1, -1, 0, [129, 64], 0),
    (1, 40, 300, 2, 1, 128, BF, 20, 3, 500, None, 250),
    (2, 9, 50, 2, 2, 64, FP, 4, 0, 2, [50, 50], [-3, 48]),
    (2, 9, 50, 2, 2, 256, BF, 4, 0, 0, [50, 50], [-20, 90]),
    (1, 700, 700, 1, 1, 64, BF, 64, 0, 0, None, 0),
    (1, 700, 700, 1, 1, 128, FP, 63, 64, 65, None, 0),
    (1, 521, 521, 2, 1, 256, BF, 100, 10, 33, None, 0),
    (2, 300, 300, 6, 2, 128, BF, 127, 0, 4, [300, 77], 0),
    (1, 517, 1030, 5, 1, 64, FP, 200, 0, 130, [1001], 513),
    (3, 193, 193, 12, 4, 64, BF, 0, 0, 0, [193, 0, 1], 0),
    (1, 333, 333, 8, 8, 128, BF, -1, 5, 0, [300], 0),
    (4, 400, 400, 8, 4, 64, BF, 32, 32, 3, [400, 399, 65, 64], 0),
    (16, 160, 160, 16, 16, 128, BF, 40, 0, 1, None, 0),
    (2, 2100, 2100, 20, 5, 64, FP, 90, 0, 4, [2100, 1500], 0),
    (1, 600, 600, 2, 2, 128, BF, 5, 0, 3, [600], [10]),
    (1, 50, 50, 71, 1, 64, BF, 9, 2, 1, None, 0),
    (2, 3, 130, 128, 1, 128, FP, 60, 0, 4, [130, 40], 100),
    (1, 35, 90, 300, 2, 64, BF, -1, 0, 0, None, 55),
]
# ... and with rows enough for shared tiles
MANY = [
    (8, 33, 33, 32, 16, 64, BF, 7, 0, 4, None, 0),
    (8, 100, 100, 16, 16, 256, FP, 16, 16, 0, None, 0),
    (8, 65, 200, 48, 16, 128, BF, 63, 0, 64, [200, 0, 1, 64, 65, 128, 199, 37], 120),
    (4, 150, 150, 60, 12, 64, BF, -1, 0, 0, None, 0),
    (8, 40, 129, 16, 16, 128, BF, -1, -1, 0, [129, 64, 0, 1, 33, 32, 31, 100], 0),
    (8, 70, 300, 32, 16, 128, FP, 20, 3, 500, None, 250),
    (8, 9, 150, 32, 32, 64, FP, 4, 0, 2, [150] * 8, [-3, 48, -20, 190, 0, 1, 149, 140]),
    (4, 270, 270, 16, 16, 256, BF, 100, 10, 33, [270, 3, 0, 200], 0),
    (64, 1, 200, 8, 4, 128, BF, 50, 0, 4, [200 - 3 * i for i in range(64)], 130),
    (1, 140, 140, 64, 64, 128, BF, 0, 0, 0, None, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,Sq,Skv,Hq,Hk,D,dtype,left,right,sinks,lens,first", CASES + MANY)
def test_forward(B, Sq, Skv, Hq, Hk, D, dtype, left, right, sinks, lens, first):
    q, k, v = tensors(B, Sq, Skv, Hq, Hk, D, dtype, Sq + Skv)
    n = [Skv] * B if lens is None else lens
    starts = first if isinstance(first, list) else [first] * B
    ref = forward(q, k, v, D ** -0.5, left, right, sinks, n, starts)
    up = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32).cuda()
    q, k, v = q.cuda(), k.cuda(), v.cuda()
    for b in range(B):
        k[b, n[b]:], v[b, n[b]:] = float("nan"), float("inf")          # padding may hold anything
    args = (q, k, v, D ** -0.5, left, right, sinks)
    o = W.sdpa_window(*args, kv_lens=up(lens), q_start=up(first) if isinstance(first, list) else first)
    assert o.shape == q.shape and o.dtype == dtype
    if isinstance(first, list):
        check_forward(o, None, ref, dtype)
    else:
        fwd = W.sdpa_window_train_fwd(*args, kv_lens=None if lens is None else up(lens).long(), q_start=first)
        check_forward(fwd.o, fwd.stats, ref, dtype)
        assert torch.equal(o, fwd.o) and fwd.stats.shape == (B, Hq, Sq, 1)
    empty = torch.isinf(ref[1]).transpose(1, 2)
    assert (o.cpu()[empty] == 0).all()


DECODE = [
    # B, Sq, capacity, Hq, Hk, D, type, left, sinks, lens
    (1, 1, 1, 1, 1, 64, BF, 0, 0, [1]),
    (1, 1, 5000, 4, 1, 128, BF, -1, 0, [4999]),
    (4, 1, 300, 8, 2, 64, FP, 63, 4, [300, 0, 1, 77]),
    (3, 4, 600, 6, 2, 128, BF, 100, 4, [600, 3, 130]),
    (2, 7, 129, 40, 5, 64, BF, -1, 0, [129, 5]),
    (2, 1, 2050, 3, 3, 256, BF, 1023, 77, [2050, 1100]),
    (1, 33, 700, 2, 1, 128, FP, 64, 1, [650]),
    (5, 1, 64, 12, 12, 128, BF, 10, 64, [64, 1, 2, 30, 11]),
    (2, 1, 200, 2, 2, 64, BF, 8, 3, [500, -4]),
    (1, 2, 9000, 16, 1, 256, FP, 8191, 4, [8999]),
    (1, 1, 6000, 8, 1, 64, FP, -1, 3, [5990]),
    (2, 1, 1500, 4, 2, 64, BF, -1, 0, [1500, 12]),
    (64, 1, 90, 8, 4, 128, FP, 40, 3, [90 - i for i in range(64)]),
    (128, 3, 70, 2, 2, 256, BF, -1, 0, [i % 71 for i in range(128)]),
    (3, 1, 700, 96, 1, 128, BF, 300, 2, [700, 299, 1]),
    (2, 2, 400, 65, 1, 256, FP, -1, 0, [400, 1]),
    (32, 1, 1100, 32, 8, 128, BF, -1, 0, [1100 - 37 * i for i in range(32)]),
    (96, 1, 1500, 8, 4, 128, FP, 1200, 4, [1500 - 15 * i for i in range(96)]),
    (33, 1, 1030, 8, 8, 128, BF, -1, 0, [1030 - 31 * i for i in range(33)]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,Sq,cap,Hq,Hk,D,dtype,left,sinks,lens", DECODE)
def test_decode(B, Sq, cap, Hq, Hk, D, dtype, left, sinks, lens):
    q, k, v = tensors(B, Sq, cap, Hq, Hk, D, dtype, cap)
    n = [min(max(x, 0), cap) for x in lens]                            # (lengths outside the cache: the nearer bound)
    ref = forward(q, k, v, D ** -0.5, left, 0, sinks, n, [x - Sq for x in n])
    kd, vd = k.cuda(), v.cuda()
    for b in range(B):
        kd[b, n[b]:], vd[b, n[b]:] = float("inf"), float("nan")
    lens = torch.tensor(lens).cuda()
    o = W.sdpa_window_decode(q.cuda(), kd, vd, lens, D ** -0.5, left, sinks)
    check_forward(o, None, ref, dtype)
    assert (o.cpu()[torch.isinf(ref[1]).transpose(1, 2)] == 0).all()
    assert torch.equal(o, W.sdpa_window_decode(q.cuda(), kd, vd, lens.int(), D ** -0.5, left, sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("Sq,first,H", [(40, 960, 2), (640, 300, 2), (300, 500, 32)])
def test_keys_that_no_query_sees_are_not_read(Sq, first, H):
    """Between the sinks and the window's left edge, behind its right edge and behind the length: whatever lies there, the same bits."""
    B, Skv, D, left, right, sinks, n = 2, 1100, 128, 50, 5, 70, 1090
    q, k, v = (t.cuda() for t in tensors(B, Sq, Skv, H, H, D, BF, 3))
    lens = torch.tensor([n, n], dtype=torch.int32).cuda()
    args = dict(scale=0.1, left=left, right=right, sinks=sinks, kv_lens=lens, q_start=first)
    want = W.sdpa_window(q, k, v, **args)
    lo, hi = first - left, min(first + Sq - 1 + right, n - 1)
    for bad in (float("nan"), float("inf"), -3e38):
        k2, v2 = k.clone(), v.clone()
        for t in (k2, v2):
            t[:, sinks:lo] = bad
            t[:, hi + 1:] = bad
        assert torch.equal(W.sdpa_window(q, k2, v2, **args), want)


@pytest.mark.gpu
@pytest.mark.parametrize("S,H,D", [(600, 1, 64), (130, 64, 64), (130, 64, 128)])
def test_extreme_scores(S, H, D):
    """Scores of +-1e4 and more, rising along the keys and falling, equal ones, and masked keys whose scores would be the largest."""
    B = 1
    q, k, v = tensors(B, S, S, H, H, D, BF, 5)
    rise = torch.linspace(-30, 30, S).view(1, S, 1, 1)
    for kk, qq in ((k * 0 + rise, q * 0 + 4), (k * 0 - rise, q * 0 + 4), (k * 0, q), (k * 40, q * 40)):
        qq, kk = qq.to(BF), kk.to(BF)
        ref = forward(qq, kk, v, 1.0, 100, 0, 2, [S], [0])
        fwd = W.sdpa_window_train_fwd(qq.cuda(), kk.cuda(), v.cuda(), 1.0, 100, 0, 2)
        check_forward(fwd.o, fwd.stats, ref, BF)


@pytest.mark.gpu
def test_layouts():
    """Parts of a joint projection, [B,H,S,D] memory, rows off 16 bytes, broadcast keys, and rows of a larger cache."""
    B, S, Hq, Hk, D = 2, 150, 4, 2, 128
    joint = torch.randn((B, S, Hq + 2 * Hk, D), generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    q, k, v = joint[:, :, :Hq], joint[:, :, Hq:Hq + Hk], joint[:, :, Hq + Hk:]
    call = lambda q, k, v: W.sdpa_window(q, k, v, 0.1, 40, 0, 4)
    want = call(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(call(q, k, v), want)
    bhsd = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(call(*bhsd), want)
    odd = [torch.empty(t.numel() + 1, dtype=BF, device="cuda")[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    assert torch.equal(call(*odd), want)
    cache = torch.full((B, 400, Hk, D), float("nan"), dtype=BF, device="cuda")
    cache[:, 100:100 + S] = k
    assert torch.equal(call(q, cache[:, 100:100 + S], v), want)
    one = k[:1].expand(B, S, Hk, D)
    assert torch.equal(call(q, one, v), call(q, one.contiguous(), v))


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """A cache whose rows lie 128 KiB apart, more than 4 GiB from first to last, and a head offset behind them."""
    n, D = 40000, 64
    wide = torch.empty((n, 65536), dtype=BF, device="cuda")
    small = torch.randn((n, 2, D), generator=torch.Generator().manual_seed(2)).to(BF)
    k = wide.as_strided((1, n, 2, D), (n * 65536, 65536, 32768, 1))
    v = wide.as_strided((1, n, 2, D), (n * 65536, 65536, 32768, 1), 128)
    k.copy_(small.cuda().view(1, n, 2, D))
    v.copy_(small.cuda().view(1, n, 2, D) * 0.5)
    q = torch.randn((1, 2, 4, D)).to(BF)
    lens = torch.tensor([n - 3]).cuda()
    ref = forward(q, k, v, 0.125, 300, 0, 4, [n - 3], [n - 5])
    check_forward(W.sdpa_window_decode(q.cuda(), k, v, lens, 0.125, 300, 4), None, ref, BF)
    q = torch.randn((1, 600, 4, D)).to(BF)
    ref = forward(q, k[:, 39000:], v[:, 39000:], 0.125, 20, 0, 0, [1000], [300])
    check_forward(W.sdpa_window(q.cuda(), k, v, 0.125, 20, 0, 0, q_start=39300), None, ref, BF)
    q = torch.randn((1, 4200, 4, D)).to(BF).cuda()
    window = (0.125, 20, 0, 4, None, 35000)
    assert torch.equal(W.sdpa_window(q, k, v, *window), W.sdpa_window(q, k.contiguous(), v.contiguous(), *window))


@pytest.mark.gpu
def test_streams_graphs_and_repeats():
    """The same bits on another stream, on every call, and from a captured graph whose lengths and inputs change between replays."""
    B, cap, Hq, Hk, D = 3, 900, 8, 2, 128
    q, k, v = (t.cuda() for t in tensors(B, 1, cap, Hq, Hk, D, BF, 8))
    qp, kp, vp = (t.cuda() for t in tensors(1, 700, 700, 4, 4, 64, BF, 9))
    lens = torch.tensor([900, 400, 17], dtype=torch.int32).cuda()
    dec = lambda: W.sdpa_window_decode(q, k, v, lens, 0.1, -1, 0)
    pre = lambda: W.sdpa_window(qp, kp, vp, 0.1, 60, 0, 2)
    want = dec(), pre()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = dec(), pre()
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs = []
    for _ in range(2):                                                 # (two graphs: each has a workspace of its own)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = dec(), pre()
        graphs.append((g, out))
    for i in range(4):
        lens.copy_(torch.tensor([900 - 13 * i, 31 * i, 500], dtype=torch.int32))
        k.copy_(torch.randn(k.shape, device="cuda"))
        qp.copy_(torch.randn(qp.shape, device="cuda"))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        eager = dec(), pre()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1]), i


def grads(q, k, v, d, *window, lens=None, first=0):
    fwd = W.sdpa_window_train_fwd(q, k, v, *window, kv_lens=lens, q_start=first)
    g = W.sdpa_window_backward(fwd, d)
    return fwd, (g.d_q, g.d_k, g.d_v)


# (the forward's cases that a backward takes, sinks that many later blocks of queries see with them, windows a little over whole tiles, and key blocks
# shared by several workgroups: few heads and long windows)
BACKWARD = [c for c in CASES if c[5] != 256 and not isinstance(c[11], list)] + [
    (1, 1500, 1500, 2, 1, 64, BF, 100, 0, 4, None, 0),
    (1, 1500, 1500, 2, 1, 128, BF, 2, 0, 130, [1490], 0),
    (2, 900, 900, 3, 3, 64, FP, 1, 1, 1, [900, 450], 0),
    (1, 1300, 1300, 1, 1, 128, FP, -1, 0, 0, None, 0),
    (1, 700, 1300, 4, 2, 64, BF, -1, 3, 0, [1300], 600),
    (1, 260, 260, 2, 2, 128, BF, 2, 0, 0, None, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,Sq,Skv,Hq,Hk,D,dtype,left,right,sinks,lens,first", BACKWARD)
def test_backward(B, Sq, Skv, Hq, Hk, D, dtype, left, right, sinks, lens, first):
    q, k, v = tensors(B, Sq, Skv, Hq, Hk, D, dtype, Sq + Skv)
    d = torch.randn(q.shape, generator=torch.Generator().manual_seed(4)).to(dtype)
    n = [Skv] * B if lens is None else lens
    ref = forward(q, k, v, D ** -0.5, left, right, sinks, n, [first] * B)
    want = backward(q, k, v, d, D ** -0.5, ref, Hq // Hk)
    kd, vd = k.cuda(), v.cuda()
    for b in range(B):
        kd[b, n[b]:], vd[b, n[b]:] = float("nan"), float("inf")
    lens = None if lens is None else torch.tensor(lens, dtype=torch.int32).cuda()
    args = (q.cuda(), kd, vd, d.cuda(), D ** -0.5, left, right, sinks)
    fwd, got = grads(*args, lens=lens, first=first)
    check_backward(got, want)
    for x, y in zip(got, grads(*args, lens=lens, first=first)[1]):
        assert torch.equal(x, y)


def test_the_gradient_formulas_against_central_differences():
    B, Sq, Skv, Hq, Hk, D = 1, 9, 11, 4, 2, 8
    g = torch.Generator().manual_seed(6)
    q, k, v, d = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((B, Sq, Hq, D), (B, Skv, Hk, D), (B, Skv, Hk, D), (B, Sq, Hq, D)))
    args = (0.5, 3, 1, 2, [10], [1])
    f = lambda *t: float((forward(*t, *args)[0] * d).sum())
    got = backward(q, k, v, d, 0.5, forward(q, k, v, *args), Hq // Hk)
    for which in range(3):
        for i in (0, 5, 37, 70, 133):
            t = [q.clone(), k.clone(), v.clone()]
            t[which].view(-1)[i] += 1e-5
            up = f(*t)
            t[which].view(-1)[i] -= 2e-5
            assert abs((up - f(*t)) / 2e-5 - float(got[which][0].reshape(-1)[i])) < 1e-8


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_backward_of_keys_that_no_query_sees(D):
    """Stale keys between the sinks and the window, and behind it, whatever they hold: zeros for them, the same bits for the rest."""
    B, Sq, Skv, H = 1, 200, 900, 2
    q, k, v = (t.cuda() for t in tensors(B, Sq, Skv, H, H, D, BF, 3))
    d = torch.randn(q.shape, device="cuda").to(BF)
    window = (0.1, 50, 5, 70)
    want = grads(q, k, v, d, *window, first=500)[1]
    k2, v2 = k.clone(), v.clone()
    for t in (k2, v2):
        t[:, 70:450], t[:, 705:] = float("nan"), float("inf")
    got = grads(q, k2, v2, d, *window, first=500)[1]
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    assert (want[1][:, 70:450] == 0).all() and (want[2][:, 705:] == 0).all()


@pytest.mark.gpu
def test_backward_layouts():
    """Parts of a joint projection and an upstream gradient of other strides, as autograd hands them over."""
    B, S, Hq, Hk, D = 2, 300, 4, 2, 128
    joint = torch.randn((B, S, Hq + 2 * Hk, D), generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    q, k, v = joint[:, :, :Hq], joint[:, :, Hq:Hq + Hk], joint[:, :, Hq + Hk:]
    d = torch.randn(q.shape, device="cuda").to(BF)
    want = grads(q.contiguous(), k.contiguous(), v.contiguous(), d, 0.1, 40, 0, 4)[1]
    for g in (d.transpose(1, 2).contiguous().transpose(1, 2), torch.empty(d.numel() + 1, dtype=BF, device="cuda")[1:].view(d.shape).copy_(d)):
        for x, y in zip(grads(q, k, v, g, 0.1, 40, 0, 4)[1], want):
            assert torch.equal(x, y)
    one = d[:, :, :, :1].expand(d.shape)                               # (a broadcast gradient: rows are not dense)
    for x, y in zip(grads(q, k, v, one, 0.1, 40)[1], grads(q, k, v, one.contiguous(), 0.1, 40)[1]):
        assert torch.equal(x, y)
    leaf = joint.clone().requires_grad_()
    att = W.record_sdpa_window(leaf[:, :, :Hq], leaf[:, :, Hq:Hq + Hk], leaf[:, :, Hq + Hk:], 0.1, 40, 0, 4)
    (g,) = torch.autograd.grad(att, leaf, d)
    for x, y in zip((g[:, :, :Hq], g[:, :, Hq:Hq + Hk], g[:, :, Hq + Hk:]), want):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_backward_captured():
    """A training step in a graph, replayed with other inputs and lengths and the program's own work in between."""
    B, S, H, D = 2, 640, 2, 64
    q, k, v = (t.cuda() for t in tensors(B, S, S, H, H, D, BF, 8))
    d = torch.randn(q.shape, device="cuda").to(BF)
    lens = torch.tensor([640, 300], dtype=torch.int32).cuda()
    step = lambda: grads(q, k, v, d, 0.1, 80, 0, 3, lens=lens)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fwd, out = step()
    for i in range(4):
        q.copy_(torch.randn(q.shape, device="cuda"))
        lens.copy_(torch.tensor([640 - i, 77 * i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want, eager = step()
        torch.cuda.synchronize()
        assert torch.equal(fwd.o, want.o) and torch.equal(fwd.stats, want.stats)
        for x, y in zip(out, eager):
            assert torch.equal(x, y), i


def test_refusals():
    q, k = torch.zeros((2, 4, 4, 64), dtype=BF), torch.zeros((2, 6, 2, 64), dtype=BF)
    lens = torch.tensor([6, 6])
    ok = dict(q=q, k=k, v=k, scale=0.1, left=3, right=0, sinks=0)
    for change, text in (
            (dict(q=q[0]), "rank-4"), (dict(v=k[:, :3]), "k/v shape"), (dict(q=q.float(), k=k.float(), v=k.float()), "BF16 or F16"), (dict(v=k.half()), "all the same"),
            (dict(q=q[:1]), "disagree"), (dict(q=q[:, :, :3]), "cannot share"), (dict(q=q[..., :32], k=k[..., :32], v=k[..., :32]), "Dh=32"),
            (dict(q=q[:, :0]), "empty"), (dict(k=k[:, :0], v=k[:, :0]), "empty"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
            (dict(scale=-1.0), "scale"), (dict(left=-2), "at least"), (dict(right=-2), "at least"), (dict(sinks=-1), "at least"),
            (dict(kv_lens=lens.float()), "kv_lens"), (dict(kv_lens=lens[:1]), "kv_lens"), (dict(q_start=lens.float()), "q_start"), (dict(), "must live on the GPU")):
        with pytest.raises(Error, match=text):
            W.sdpa_window(**{**ok, **change})
    with pytest.raises(Error, match="must be an int"):
        W.sdpa_window_train_fwd(**ok, q_start=lens)
    dec = dict(q=q, k_cache=k, v_cache=k, kv_lens=lens, scale=0.1, left=3)
    for change, text in ((dict(kv_lens=None), "kv_lens"), (dict(kv_lens=lens[:1]), "kv_lens"), (dict(left=-2), "at least"), (dict(v_cache=k[:, :2]), "k/v shape"),
                         (dict(), "must live on the GPU")):
        with pytest.raises(Error, match=text):
            W.sdpa_window_decode(**{**dec, **change})
    fwd = W.SdpaWindowFwd(q, q, torch.zeros((2, 4, 4, 1)), q, k, k, 0.1, 3, 0, 0, None, 0)
    for change, d, text in ((dict(), q.half(), "type of the forward"), (dict(), q[:, :3], "does not match"), (dict(stats=torch.zeros(3)), q, "stats must be"),
                            (dict(q=q.repeat(1, 1, 1, 4), k=k.repeat(1, 1, 1, 4), v=k.repeat(1, 1, 1, 4)), q, "Dh=256"), (dict(), q, "must live on the GPU")):
        with pytest.raises(Error, match=text):
            W.sdpa_window_backward(W.SdpaWindowFwd(**{**fwd.__dict__, **change}), d)


def test_c_refusals():
    """Codes for arguments that never reach a device (addresses are made up and not read)."""
    import ctypes
    from mojodiffusion_amd import _lib
    L = _lib.lib()
    A = 1 << 20
    st = _lib.strides_bhnd(8, 4, 64)
    S = lambda *s: (ctypes.c_int64 * 4)(*s)
    base = dict(q=A, k=A, v=A, o=A, B=1, Hq=4, Hk=4, Nq=8, Nkv=8, D=64, type=0, scale=0.1, qs=st, ks=st, vs=st, os=st, off=(0, 0, 0, 0), left=3, right=0,
                sinks=0, start=0, ws=None, nws=0)

    def call(**change):
        a = {**base, **change}
        return L.mi355_sage_sdpa_window(a["q"], a["k"], a["v"], a["o"], None, None, a["B"], a["Hq"], a["Hk"], a["Nq"], a["Nkv"], a["D"], a["type"], a["scale"],
                                        a["qs"], a["ks"], a["vs"], a["os"], *a["off"], 0, a["left"], a["right"], a["sinks"], None, None, a["start"], None,
                                        a["ws"], a["nws"])
    for change in (dict(q=None), dict(o=None), dict(vs=None), dict(B=0), dict(Hk=0), dict(Hq=6), dict(Nq=0), dict(Nkv=-1), dict(scale=0.0), dict(scale=float("inf")),
                   dict(scale=float("nan")), dict(left=-2), dict(right=-2), dict(sinks=-1), dict(os=S(0, 0, 64, 1)), dict(os=S(0, 512, 0, 1))):
        assert call(**change) == -1, change
    for change in (dict(D=96), dict(type=2), dict(Nq=1 << 29), dict(Nkv=(1 << 29) + 1), dict(start=(1 << 29) + 1), dict(ks=S(0, 64, 256, 2)),
                   dict(qs=S(0, 60, 256, 1)), dict(k=A + 8), dict(off=(0, 0, 4, 0)), dict(ks=S(0, 64, 1 << 26, 1)), dict(vs=S(0, 64, -64, 1)),
                   dict(Hk=1, qs=S(0, 1 << 31, 64, 1)), dict(B=1 << 16, Hq=1 << 12, Hk=1 << 12, Nq=64)):
        assert call(**change) == -2, change
    assert call(Nkv=8192, left=-1, ws=A, nws=8) == -3 and call(Nkv=8192, left=-1, ws=A + 8, nws=1 << 30) == -3
    assert L.mi355_sage_window_workspace_bytes(1, 4, 4, 8, 8192, 64, -1, 0, 0) > 1000
    assert L.mi355_sage_window_workspace_bytes(1, 4, 3, 8, 8192, 64, -1, 0, 0) == 0
    assert L.mi355_sage_sdpa_window_decode(A, A, A, A, 1, 4, 4, 1, 8, 64, 0, 0.1, st, st, st, st, 0, 0, 0, 0, 3, 0, None, None, None, 0) == -1
    bwd = [A] * 10 + [1, 4, 4, 8, 8, 64, 0, 0.1] + [st] * 8 + [0] * 9 + [3, 0, 0, None, 0, None]
    assert L.mi355_sage_sdpa_window_bwd(*bwd, A, 8) == -3
    for at, value, code in ((0, None, -1), (9, None, -1), (18, None, -1), (15, 256, -2), (11, 5, -1), (16, 2, -2), (22, off_rows(S), -2), (25, S(0, 64, 256, 2), -2),
                            (23, S(0, 0, 64, 1), -1), (24, S(0, 64, 0, 1), -1), (25, S(0, 0, 64, 1), -1)):
        args = list(bwd)
        args[at] = value
        assert L.mi355_sage_sdpa_window_bwd(*args, A, 1 << 30) == code, at
    assert L.mi355_sage_window_bwd_workspace_bytes(1, 4, 4, 8, 8, 256, 3, 0, 0) == 0
    assert L.mi355_sage_window_bwd_workspace_bytes(1, 4, 2, 8, 8, 64, 3, 0, 0) > 0


def off_rows(S):
    return S(0, 60, 256, 1)
