"""Attention through a window in float64, from the definition, and the bounds that go with it."""
import torch


def visible(p, n, Skv, left, right, sinks):
    """[len(p), Skv]: which keys of a sequence of n the queries at positions p see."""
    p, j = p.view(-1, 1), torch.arange(Skv).view(1, -1)
    seen = j < n
    if right >= 0:
        seen = seen & (j <= p + right)
    if left >= 0:
        seen = seen & ((j >= p - left) | (j < sinks))
    return seen


def forward(q, k, v, scale, left, right, sinks, lens, starts):
    """O, L (-inf: nothing seen) and the bounds' sizes, float64 on the CPU.

    Bounds.  u = eps / 2 of the type.  A score is a sum of D products in fp32: off by at most delta = scale D 2^-24 sum |q||k| (and a
    few steps of its own for the scale and the reference: 2^-22 of |S| + |L|), which changes a weight by as much, relatively.  A weight is rounded
    to the type (u), products and sums over n keys are fp32 (n 2^-24 relative to sum w|v|), and O is rounded (u |O|).  fp16 weights below 2^-14 of the
    reference's have an absolute step, 2^-25 at most each; the reference's own weight is 1 or more."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    B, Sq, Hq, D = q.shape
    Skv, g = k.shape[1], Hq // k.shape[2]
    O, L = torch.zeros_like(q), torch.full((B, Hq, Sq), -torch.inf, dtype=torch.float64)
    W, A, E = torch.zeros((B, Hq, Sq, Skv), dtype=torch.float64), torch.zeros_like(q), torch.zeros((B, Hq, Sq), dtype=torch.float64)
    F = torch.zeros_like(q)
    for b in range(B):
        seen = visible(starts[b] + torch.arange(Sq), lens[b], Skv, left, right, sinks)
        some = seen.any(1)
        for h in range(Hq):
            # (rows of padding are not part of anything)
            kk, vv = k[b, :, h // g].masked_fill(~seen.any(0).view(-1, 1), 0.0), v[b, :, h // g].masked_fill(~seen.any(0).view(-1, 1), 0.0)
            s = (q[b, :, h] @ kk.T * scale).masked_fill(~seen, -torch.inf)
            L[b, h] = torch.logsumexp(s, 1)
            W[b, h] = torch.where(some.view(-1, 1), torch.exp(s - torch.where(some, L[b, h], 0.0).view(-1, 1)), 0.0)
            O[b, :, h], A[b, :, h] = W[b, h] @ vv, W[b, h] @ vv.abs()
            F[b, :, h] = seen.double() @ vv.abs()
            size = (q[b, :, h].abs() @ kk.abs().T * scale).masked_fill(~seen, 0.0).amax(1)
            E[b, h] = size * D * 2.0 ** -24 + 2.0 ** -22 * (size + torch.where(some, L[b, h].abs(), 0.0) + 1)
    return O, L, W, A, F, E


def check_forward(o, stats, ref, dtype):
    O, L, W, A, F, E = ref
    u, n = torch.finfo(dtype).eps / 2, W.shape[3]
    e = E.transpose(1, 2).unsqueeze(-1)
    bound = u * O.abs() + A * (1.01 * u + n * 2.0 ** -24 + 2.1 * e) + (F * 2.0 ** -25 if dtype == torch.float16 else 0) + 1e-30
    err = (o.double().cpu() - O).abs()
    assert torch.isfinite(o).all() and (err <= bound).all(), float((err / bound).max())
    if stats is not None:
        got = stats.double().cpu().reshape(L.shape)
        empty = torch.isinf(L)
        assert torch.equal(torch.isinf(got), empty) and (got[empty] < 0).all()
        assert ((got - L).abs() <= E + n * 2.0 ** -24)[~empty].all()


def backward(q, k, v, d, scale, ref, g):
    """Gradients by the formulas and the sizes of their bounds, float64; ref: forward's result, g: query heads to a key head.

    Bounds.  dS = P (dP - Delta).  P: recomputed from scores and a statistic that are off by E each (2 E relative), rounded to the type (u) for dV, handed on
    with 11 bits (2^-10) and, as part of dS, rounded (u) for dQ and dK.  Delta is a product with O, stored to twice the type's bits and else off
    by the forward's bound: dDelta = sum |dO| bound(O).  dP and Delta are fp32 sums of D products (D 2^-24 of their sizes).  Every sum over rows or keys is fp32, and
    the result is rounded (u).  dQ is taken as scale dS (K - c), c a mean of keys: an error of dS meets |k| + |c|, and |c| is no larger than a key.  F: what fp16 loses below its normal range, 2^-25 for every P and dS."""
    O, L, W, A, F, E = ref
    dtype = q.dtype
    u = torch.finfo(dtype).eps / 2
    q, k, v, d = (t.double().cpu() for t in (q, k, v, d))
    B, Sq, Hq, D = q.shape
    n = max(Sq * g, k.shape[1])
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    bq, bk, bv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    e = E.transpose(1, 2).unsqueeze(-1)
    bo = 2 * u * u * O.abs() + A * (1.01 * u + W.shape[3] * 2.0 ** -24 + 2.1 * e) + (F * 2.0 ** -25 if dtype == torch.float16 else 0)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for b in range(B):
        for h in range(Hq):
            w, ww = W[b, h], (W[b, h] > 0).double()
            used = (ww.sum(0) > 0).view(-1, 1)
            qh, dh = q[b, :, h], d[b, :, h]
            kh, vh = k[b, :, h // g].masked_fill(~used, 0.0), v[b, :, h // g].masked_fill(~used, 0.0)
            dp = dh @ vh.T
            delta = (w * dp).sum(1, keepdim=True)
            ds = w * (dp - delta)
            dp_size = dh.abs() @ vh.abs().T + (dh.abs() * O[b, :, h].abs()).sum(1, keepdim=True)
            d_delta = (dh.abs() * bo[b, :, h]).sum(1, keepdim=True) + D * 2.0 ** -24 * dp_size
            p_err = (2.2 * E[b, h].view(-1, 1) + n * 2.0 ** -24) * w
            ds_err = ds.abs() * (1.01 * u + 2.0 ** -10) + (dp - delta).abs() * (p_err + tiny) + 1.01 * (w + tiny) * d_delta + tiny * ww
            dq[b, :, h] = scale * ds @ kh
            bq[b, :, h] = scale * (ds_err + n * 2.0 ** -24 * ds.abs()) @ (kh.abs() + kh.abs().amax(0))
            dk[b, :, h // g] += scale * ds.T @ qh
            bk[b, :, h // g] += scale * (ds_err + n * 2.0 ** -24 * ds.abs()).T @ qh.abs()
            dv[b, :, h // g] += w.T @ dh
            bv[b, :, h // g] += (w * (1.01 * u + n * 2.0 ** -24) + p_err + tiny * ww).T @ dh.abs()
    return tuple((x, u * x.abs() + 1.01 * y + tiny) for x, y in ((dq, bq), (dk, bk), (dv, bv)))


def check_backward(got, want):
    for name, x, (ref, bound) in zip(("dQ", "dK", "dV"), got, want):
        err = (x.double().cpu() - ref).abs()
        assert torch.isfinite(x).all() and (err <= bound + 1e-30).all(), (name, float((err / (bound + 1e-30)).max()))
