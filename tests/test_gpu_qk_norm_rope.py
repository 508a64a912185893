"""qk_norm_rope and its gradient against the formulas in float64.

Tolerances.  Everything between the rows read and the rows written is fp32: a row's sum of D <= 256 squares takes
16 + log2(16) additions per lane and tree (relative error < 24 * 2^-24), the root and the quotient 2 more steps, the products
with r, g, cos and sin one each, so a rotated channel is off by less than 2^-19 of |y_a| + |y_b|, the two values it is made
of.  On top comes the one rounding to the stored type, eps / 2 of the value (2^-25 where fp16 has run out of exponents)."""
import pytest
import torch

from mojodiffusion_amd import norm_rope as N
from mojodiffusion_amd.attention_sage import Error

F32 = 2.0 ** -19


def tables(rows, rot, dtype=torch.float32, device="cpu"):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / rot)
    return angle.cos().to(dtype).to(device), angle.sin().to(dtype).to(device)


def pairs(rot, halfsplit):
    i = torch.arange(rot // 2)
    return (i, i + rot // 2) if halfsplit else (2 * i, 2 * i + 1)


def reference(x, gain, eps, cos, sin, halfsplit, rows):
    """z, and the bound's |y_a| + |y_b|, in float64; cos/sin [P, rot/2] or None, rows [B,S]."""
    x, gain = x.double(), gain.double()
    y = x * gain / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    z, size = y.clone(), y.abs()
    if cos is not None:
        a, b = pairs(2 * cos.shape[1], halfsplit)
        c, s = cos.double()[rows].unsqueeze(2), sin.double()[rows].unsqueeze(2)
        z[..., a], z[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
        both = y[..., a].abs() + y[..., b].abs()
        size = size.clone()
        size[..., a], size[..., b] = both, both
    return z, size


def rounding(t):
    return torch.finfo(t).eps / 2, {torch.float16: 2.0 ** -25}.get(t, 1e-38)


def close(got, want, slack):
    rel, tiny = rounding(got.dtype)
    err = (got.double().cpu() - want).abs()
    bound = rel * (want.abs() + slack) + tiny + slack
    assert torch.isfinite(got).all() and (err <= bound).all(), float((err / bound).max())


def inputs(B, S, Hq, Hk, D, dtype, seed, gain_dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn((B, S, Hq + 2 * Hk, D), generator=g).to(dtype)
    gains = [(1 + 0.3 * torch.randn(D, generator=g)).to(gain_dtype) for _ in range(2)]
    return qkv, gains


# head dims with every number of lanes to a row, partly filled ones among them; rotated all, a part, nothing; one token, odd counts,
# enough rows for both forms of the launch (few rows: one head to a group of lanes; more: four share their tables)
CASES = [
    (1, 1, 1, 1, 64, 64, torch.bfloat16), (3, 5, 7, 2, 64, 32, torch.float16), (2, 17, 5, 5, 128, 128, torch.float32),
    (1, 33, 3, 1, 256, 64, torch.bfloat16), (2, 9, 4, 3, 96, 96, torch.float16), (1, 7, 2, 2, 16, 16, torch.float32),
    (2, 11, 6, 1, 80, 48, torch.bfloat16), (1, 13, 3, 3, 192, 0, torch.float16), (1, 1153, 48, 12, 128, 128, torch.bfloat16),
    (2, 2311, 18, 6, 64, 64, torch.float16), (1, 1601, 15, 5, 256, 128, torch.float32), (5, 1, 48, 12, 128, 64, torch.bfloat16),
    (1, 4096, 30, 2, 144, 144, torch.bfloat16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("halfsplit", [False, True])
@pytest.mark.parametrize("B,S,Hq,Hk,D,rot,dtype", CASES)
def test_forward(B, S, Hq, Hk, D, rot, dtype, halfsplit):
    tdt = torch.bfloat16 if S % 2 else torch.float32
    qkv, (gq, gk) = inputs(B, S, Hq, Hk, D, dtype, 7 * S + D, torch.float32 if halfsplit else dtype)
    dev = qkv.cuda()
    q, k = dev[:, :, :Hq], dev[:, :, Hq:Hq + Hk]                  # the projection's own layout
    cos, sin = tables(S, rot, tdt) if rot else (None, None)
    up = lambda t: None if t is None else t.cuda()
    got = N.qk_norm_rope(q, k, gq.cuda(), gk.cuda(), 1e-6, up(cos), up(sin), halfsplit)
    rows = torch.arange(S).expand(B, S)
    for y, x, g in ((got[0], qkv[:, :, :Hq], gq), (got[1], qkv[:, :, Hq:Hq + Hk], gk)):
        assert y.dtype == dtype and y.is_contiguous()
        want, size = reference(x, g, 1e-6, cos, sin, halfsplit, rows)
        close(y, want, F32 * size)


@pytest.mark.gpu
@pytest.mark.parametrize("ptype,shape", [(torch.int32, "BS"), (torch.int64, "BS"), (torch.int64, "S"), (torch.int32, "1S")])
def test_positions(ptype, shape):
    B, S, Hq, Hk, D = 3, 19, 4, 2, 128
    qkv, (gq, gk) = inputs(B, S, Hq, Hk, D, torch.bfloat16, 3)
    cos, sin = tables(40000, D)
    pos = torch.randint(0, 40000, (B if shape == "BS" else 1, S), generator=torch.Generator().manual_seed(1))
    pos[0, 3] = pos[0, 4]                                         # the same row twice
    pos[0, 0], pos[0, 1] = 0, 39999
    arg = (pos[0] if shape == "S" else pos).to(ptype).cuda()
    dev = qkv.cuda()
    q, k = dev[:, :, :Hq], dev[:, :, Hq:Hq + Hk]
    got = N.qk_norm_rope(q, k, gq.cuda(), gk.cuda(), 1e-5, cos.cuda(), sin.cuda(), True, arg)
    want, size = reference(qkv[:, :, :Hq], gq, 1e-5, cos, sin, True, pos.expand(B, S))
    close(got[0], want, F32 * size)
    # a positions tensor of any strides
    wide = torch.stack((arg, arg), dim=-1)[..., 0]
    again = N.qk_norm_rope(q, k, gq.cuda(), gk.cuda(), 1e-5, cos.cuda(), sin.cuda(), True, wide)
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


@pytest.mark.gpu
def test_position_outside_the_tables():
    """Such a token's rotated channels are NaN, the others and all other tokens are as they are without it."""
    B, S, H, D, rot = 1, 6, 3, 64, 32
    qkv, (gq, gk) = inputs(B, S, H, H, D, torch.bfloat16, 5)
    cos, sin = (t.cuda() for t in tables(8, rot))
    dev = qkv.cuda()
    q, k = dev[:, :, :H].contiguous(), dev[:, :, H:2 * H].contiguous()
    pos = torch.tensor([[0, 1, 8, -1, 4, 2 ** 40]]).cuda()
    good = torch.tensor([[0, 1, 2, 3, 4, 5]]).cuda()
    got = N.qk_norm_rope(q, k, gq.cuda(), gk.cuda(), 1e-6, cos, sin, False, pos)
    ref = N.qk_norm_rope(q, k, gq.cuda(), gk.cuda(), 1e-6, cos, sin, False, good)
    for y, r in zip(got, ref):
        assert torch.isnan(y[:, [2, 3, 5], :, :rot]).all()
        assert torch.equal(y[:, [0, 1, 4]], r[:, [0, 1, 4]]) and torch.equal(y[..., rot:], r[..., rot:])


@pytest.mark.gpu
def test_per_head_tables_of_the_fused_call():
    """Tables of S*H rows with every row H times (what the fused attention call takes): a strided view of them is enough."""
    B, S, H, D = 2, 37, 4, 128
    qkv, (gq, gk) = inputs(B, S, H, H, D, torch.bfloat16, 9)
    cos, sin = (t.cuda() for t in tables(S, D))
    tall = [t.repeat_interleave(H, dim=0) for t in (cos, sin)]
    dev = qkv.cuda()
    args = (dev[:, :, :H], dev[:, :, H:2 * H], gq.cuda(), gk.cuda(), 1e-6)
    a, b = N.qk_norm_rope(*args, cos, sin), N.qk_norm_rope(*args, tall[0][::H], tall[1][::H])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_layouts_and_outputs(dtype):
    """[B,H,S,D] memory, rows that start off 16 bytes, in place, into a cache; everything around the written rows stays."""
    B, S, Hq, Hk, D = 2, 21, 6, 2, 128
    qkv, (gq, gk) = inputs(B, S, Hq, Hk, D, dtype, 11)
    cos, sin = (t.cuda() for t in tables(S, D))
    q, k = qkv[:, :, :Hq].contiguous().cuda(), qkv[:, :, Hq:Hq + Hk].contiguous().cuda()
    gq, gk = gq.cuda(), gk.cuda()
    want = N.qk_norm_rope(q, k, gq, gk, 1e-6, cos, sin)
    bhsd = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k)]
    odd = [torch.empty(t.numel() + 1, dtype=dtype, device="cuda")[1:].view(t.shape).copy_(t) for t in (q, k)]
    for x, y in (bhsd, odd):
        got = N.qk_norm_rope(x, y, gq, gk, 1e-6, cos, sin)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    cache = torch.full((B, 64, Hk, D), 7.0, dtype=dtype, device="cuda")
    x = q.clone()
    got = N.qk_norm_rope(x, k, gq, gk, 1e-6, cos, sin, q_out=x, k_out=cache[:, 30:30 + S])
    assert got[0] is x and torch.equal(x, want[0]) and torch.equal(cache[:, 30:30 + S], want[1])
    assert (cache[:, :30] == 7).all() and (cache[:, 30 + S:] == 7).all()


@pytest.mark.gpu
def test_degenerate_rows():
    """Rows of zeros, of the largest values whose squares fp32 holds, a NaN and an infinity: each stays in its own row."""
    D = 128
    x = torch.ones((1, 6, 1, D), dtype=torch.float32)
    x[0, 0], x[0, 1], x[0, 2] = 0, 1e18, 1e-30
    x[0, 3, 0, 5], x[0, 4, 0, 7] = float("nan"), float("inf")
    cos, sin = tables(6, D)
    one = torch.ones(D)
    q, k = N.qk_norm_rope(x.cuda(), x.cuda(), one.cuda(), one.cuda(), 1e-6, cos.cuda(), sin.cuda())
    want, size = reference(x, one, 1e-6, cos, sin, False, torch.arange(6).expand(1, 6))
    for y in (q, k):
        close(y[:, [0, 1, 2, 5]], want[:, [0, 1, 2, 5]], F32 * size[:, [0, 1, 2, 5]])
        assert torch.isnan(y[0, 3]).all() and torch.isnan(y[0, 4]).any()


def grad_reference(x, gain, d, eps, cos, sin, halfsplit, rows):
    """dx, dgain, and sizes for their bounds, in float64, from the formulas (not by automatic differentiation)."""
    x, gain, d = x.double(), gain.double(), d.double()
    D = x.shape[-1]
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    dy, size = d.clone(), d.abs()
    if cos is not None:
        a, b = pairs(2 * cos.shape[1], halfsplit)
        c, s = cos.double()[rows].unsqueeze(2), sin.double()[rows].unsqueeze(2)
        dy[..., a], dy[..., b] = d[..., a] * c + d[..., b] * s, d[..., b] * c - d[..., a] * s
        both = d[..., a].abs() + d[..., b].abs()
        size[..., a], size[..., b] = both, both
    u, xh = dy * gain, x * r
    dx = r * (u - xh * (u * xh).mean(-1, keepdim=True))
    usize = size * gain.abs()
    xsize = r * (usize + xh.abs() * (usize * xh.abs()).mean(-1, keepdim=True))
    return dx, (dy * xh).sum((0, 1, 2)), xsize, (size * xh.abs()).sum((0, 1, 2))


def test_the_gradient_formula_against_automatic_and_central_differences():
    B, S, H, D, rot = 1, 3, 2, 32, 16
    for halfsplit in (False, True):
        qkv, (g, _) = inputs(B, S, H, H, D, torch.float64, 21, torch.float64)
        x = qkv[:, :, :H].clone().requires_grad_()
        gain = g.clone().requires_grad_()
        d = torch.randn(x.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(2))
        cos, sin = tables(S, rot, torch.float64)
        rows = torch.arange(S).expand(B, S)
        f = lambda xx, gg: (reference(xx, gg, 1e-2, cos, sin, halfsplit, rows)[0] * d).sum()
        auto = torch.autograd.grad(f(x, gain), (x, gain))
        dx, dg, _, _ = grad_reference(x.detach(), g, d, 1e-2, cos, sin, halfsplit, rows)
        assert torch.allclose(auto[0], dx, rtol=1e-10, atol=1e-12) and torch.allclose(auto[1], dg, rtol=1e-10, atol=1e-12)
        h = 1e-5
        for i in (0, 17, 77, 150):
            e = torch.zeros(x.numel(), dtype=torch.float64)
            e[i] = h
            e = e.view(x.shape)
            diff = (f(x.detach() + e, g) - f(x.detach() - e, g)) / (2 * h)
            assert abs(float(diff - dx.reshape(-1)[i])) < 1e-7


@pytest.mark.gpu
@pytest.mark.parametrize("halfsplit", [False, True])
@pytest.mark.parametrize("B,S,Hq,Hk,D,rot,dtype", CASES)
def test_backward(B, S, Hq, Hk, D, rot, dtype, halfsplit):
    """dx as the forward's bound (one more mean over the row: 2^-18); a gain's gradient is a sum of n terms, in fp32 over a lane's
    rows (at most 1 + 2 n / 8192 of them, two heads a step) and 11 levels of a tree, in double above: 2^-24 per addition."""
    tdt = torch.bfloat16 if S % 2 else torch.float32
    qkv, (gq, gk) = inputs(B, S, Hq, Hk, D, dtype, 5 * S + D, torch.float32 if halfsplit else dtype)
    gen = torch.Generator().manual_seed(13)
    dq, dk = (torch.randn((B, S, h, D), generator=gen).to(dtype) for h in (Hq, Hk))
    cos, sin = tables(S, rot, tdt) if rot else (None, None)
    up = lambda t: None if t is None else t.cuda()
    dev = qkv.cuda()
    call = lambda: N.qk_norm_rope_backward(dq.cuda(), dk.cuda(), dev[:, :, :Hq], dev[:, :, Hq:Hq + Hk], gq.cuda(), gk.cuda(), 1e-6,
                                           up(cos), up(sin), halfsplit)
    got, again = call(), call()
    rows = torch.arange(S).expand(B, S)
    for y, yg, x, g, d in ((got.d_q, got.d_q_norm, qkv[:, :, :Hq], gq, dq), (got.d_k, got.d_k_norm, qkv[:, :, Hq:Hq + Hk], gk, dk)):
        dx, dg, xsize, gsize = grad_reference(x, g, d, 1e-6, cos, sin, halfsplit, rows)
        close(y, dx, 2 * F32 * xsize)
        assert yg.dtype == torch.float32
        steps = 3 + 4 * d.numel() // D // 4096 + 16
        assert ((yg.double().cpu() - dg).abs() <= (steps * 2.0 ** -24 + F32) * gsize + 2.0 ** -24 * dg.abs()).all()
    for a, b in ((got.d_q, again.d_q), (got.d_k, again.d_k), (got.d_q_norm, again.d_q_norm), (got.d_k_norm, again.d_k_norm)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_recorded_node():
    B, S, Hq, Hk, D = 2, 31, 4, 2, 64
    qkv, (gq, gk) = inputs(B, S, Hq, Hk, D, torch.bfloat16, 17, torch.bfloat16)
    cos, sin = (t.cuda() for t in tables(S, D))
    joint = qkv.cuda().requires_grad_()                          # one leaf behind both inputs
    gains = [g.cuda().requires_grad_() for g in (gq, gk)]
    q, k = joint[:, :, :Hq], joint[:, :, Hq:Hq + Hk]
    qo, ko = N.record_qk_norm_rope(q, k, *gains, 1e-6, cos, sin)
    d = [torch.randn(t.shape, device="cuda").to(t.dtype) for t in (qo, ko)]
    got = torch.autograd.grad((qo, ko), (joint, *gains), d)
    ref = N.qk_norm_rope_backward(*d, q.detach(), k.detach(), gains[0].detach(), gains[1].detach(), 1e-6, cos, sin)
    assert torch.equal(got[0][:, :, :Hq], ref.d_q) and torch.equal(got[0][:, :, Hq:Hq + Hk], ref.d_k) and (got[0][:, :, Hq + Hk:] == 0).all()
    assert torch.equal(got[1], ref.d_q_norm.to(torch.bfloat16)) and torch.equal(got[2], ref.d_k_norm.to(torch.bfloat16))


@pytest.mark.gpu
def test_streams_and_graphs():
    """On a stream of its own, and captured (forward and backward) and replayed with the program's own work in between."""
    B, S, Hq, Hk, D = 1, 257, 6, 3, 128
    qkv, (gq, gk) = inputs(B, S, Hq, Hk, D, torch.bfloat16, 23)
    cos, sin = (t.cuda() for t in tables(S, D))
    dev, gq, gk = qkv.cuda(), gq.cuda(), gk.cuda()
    q, k = dev[:, :, :Hq].contiguous(), dev[:, :, Hq:Hq + Hk].contiguous()
    fwd = lambda: N.qk_norm_rope(q, k, gq, gk, 1e-6, cos, sin)
    bwd = lambda y: N.qk_norm_rope_backward(y[0], y[1], q, k, gq, gk, 1e-6, cos, sin)
    want = fwd()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fwd()
        bwd(got)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fwd()
        g = bwd(y)
    for i in range(4):
        q.copy_(torch.randn(q.shape, device="cuda"))
        graph.replay()
        eager = fwd()
        ge = bwd(eager)
        torch.cuda.synchronize()
        assert torch.equal(y[0], eager[0]) and torch.equal(g.d_q, ge.d_q) and torch.equal(g.d_q_norm, ge.d_q_norm), i


def test_refusals():
    q, k, g = torch.zeros((1, 4, 2, 64), dtype=torch.bfloat16), torch.zeros((1, 4, 1, 64), dtype=torch.bfloat16), torch.ones(64)
    c, s = tables(4, 64)
    ok = dict(q=q, k=k, q_norm=g, k_norm=g, eps=1e-6, cos=c, sin=s)
    pos = torch.zeros((1, 4), dtype=torch.int64)
    for change, text in (
            (dict(q=q[0]), "rank-4"), (dict(q=q.double(), k=k.double()), "BF16, F16 or F32"), (dict(k=k.half()), "both the same"),
            (dict(k=k[:, :3]), "disagree"), (dict(q=q[..., :40], k=k[..., :40], q_norm=g[:40], k_norm=g[:40]), "Dh=40"),
            (dict(q_norm=torch.ones(32)), r"weight must be \[64\]"), (dict(k_norm=g.half()), "both the same"), (dict(sin=None), "come together"),
            (dict(cos=c[:3], sin=s[:3]), "3 rows for 4"), (dict(cos=c[:, :20], sin=s[:, :20]), "40 rotated"), (dict(cos=c.double(), sin=s.double()), "tables must be"),
            (dict(positions=pos.float()), "int32 or int64"), (dict(positions=pos[:, :3]), "int32 or int64"),
            (dict(positions=pos, cos=None, sin=None), "without tables"), (dict(eps=-1.0), "negative"), (dict(eps=float("nan")), "negative"),
            (dict(q=q[:, :0], k=k[:, :0]), "empty"), (dict(), "must live on the GPU")):
        with pytest.raises(Error, match=text):
            N.qk_norm_rope(**{**ok, **change})
        with pytest.raises(Error, match=text):
            N.qk_norm_rope_backward(torch.zeros_like(q), torch.zeros_like(k), **{**ok, **change})


def test_c_refusals():
    """Codes of the C entry points for arguments that never reach a device (addresses are made up and not read)."""
    import ctypes
    from mojodiffusion_amd import _lib
    L = _lib.lib()
    A = 1 << 20
    st = _lib.strides_bhnd(8, 4, 64)
    bad = (ctypes.c_int64 * 4)(8 * 4 * 64, 64, 4 * 64, 2)
    off = (ctypes.c_int64 * 4)(8 * 4 * 64, 60, 4 * 64, 1)
    flat = (ctypes.c_int64 * 4)(8 * 4 * 64, 0, 4 * 64, 1)
    base = dict(q=A, k=A, qo=A, ko=A, B=1, S=8, Hq=4, Hk=4, D=64, type=0, qs=st, ks=st, qos=st, kos=st, o=(0, 0, 0, 0), gq=A, gk=A, gt=2,
                eps=1e-6, c=A, s=A, tt=2, rot=64, rows=8, stride=32, half=0, pos=None, ps=0, pb=0)

    def fwd(**change):
        a = {**base, **change}
        return L.mi355_sage_qk_norm_rope(a["q"], a["k"], a["qo"], a["ko"], a["B"], a["S"], a["Hq"], a["Hk"], a["D"], a["type"], a["qs"], a["ks"],
                                         a["qos"], a["kos"], *a["o"], a["gq"], a["gk"], a["gt"], a["eps"], a["c"], a["s"], a["tt"], a["rot"],
                                         a["rows"], a["stride"], a["half"], a["pos"], a["ps"], a["pb"], None)
    for change in (dict(q=None), dict(ko=None), dict(gq=None), dict(qs=None), dict(B=0), dict(S=-1), dict(Hk=0), dict(type=3), dict(gt=-1), dict(tt=5),
                   dict(rot=80), dict(rot=-16), dict(c=None), dict(rows=7), dict(rows=0, pos=A, pb=4), dict(pos=A, pb=2), dict(eps=-1.0),
                   dict(kos=flat), dict(qos=flat)):
        assert fwd(**change) == -1, change
    for change in (dict(D=72, rot=32), dict(D=272), dict(rot=24), dict(qs=bad), dict(kos=off), dict(q=A + 8), dict(o=(4, 0, 0, 0)), dict(gk=A + 4),
                   dict(stride=33), dict(B=1 << 15, S=1 << 15, rows=1 << 15)):
        assert fwd(**change) == -2, change
    assert L.mi355_sage_qk_norm_rope_bwd_workspace_bytes(1, 8, 4, 4, 64) >= 2 * 64 * 4
    assert L.mi355_sage_qk_norm_rope_bwd_workspace_bytes(1, 8, 4, 4, 72) == 0
    args = [A] * 8 + [1, 8, 4, 4, 64, 0] + [st] * 6 + [0] * 6 + [A, A, 2, 1e-6, A, A, 2, 64, 8, 32, 0, None, 0, 0, None]
    assert L.mi355_sage_qk_norm_rope_bwd(*args, A, 8) == -3 and L.mi355_sage_qk_norm_rope_bwd(*args, A + 8, 1 << 20) == -3
    args[6] = None
    assert L.mi355_sage_qk_norm_rope_bwd(*args, A, 1 << 20) == -1
