"""Norm, rotation and windowed attention together, as a text model's layer uses them: a training step through both recorded nodes, and a
prompt followed by single tokens against a cache.  Every stage is checked against float64 at the inputs it was given (the bounds of
test_gpu_qk_norm_rope and window_reference), and the run against the stages called one after the other."""
import threading

import pytest
import torch

from mojodiffusion_amd import _lib
from mojodiffusion_amd import attention_window as W
from mojodiffusion_amd import norm_rope as N
from mojodiffusion_amd.attention_sage import Error
from test_gpu_qk_norm_rope import F32, close, reference, tables
from window_reference import backward, check_backward, check_forward, forward

BF = torch.bfloat16
EPS = 1e-6


def layer(B, S, Hq, Hk, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    joint = torch.randn((B, S, Hq + 2 * Hk, D), generator=g).to(dtype).cuda()
    gains = [(1 + 0.3 * torch.randn(D, generator=g)).cuda() for _ in range(2)]
    return joint, gains


def parts(joint, Hq, Hk):
    return joint[:, :, :Hq], joint[:, :, Hq:Hq + Hk], joint[:, :, Hq + Hk:]


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,Hq,Hk,D,dtype,left,sinks,lens,halfsplit", [
    (2, 333, 6, 2, 64, BF, 100, 4, [333, 200], True), (1, 150, 4, 4, 128, torch.float16, 20, 0, None, False), (3, 70, 3, 1, 128, BF, -1, 0, [70, 1, 0], False)])
def test_a_training_step(B, S, Hq, Hk, D, dtype, left, sinks, lens, halfsplit):
    joint, gains = layer(B, S, Hq, Hk, D, dtype)
    cos, sin = (t.cuda() for t in tables(S, D // 2))                   # (half of the channels are rotated)
    n = None if lens is None else torch.tensor(lens).cuda()
    leaf, gq, gk = joint.clone().requires_grad_(), gains[0].clone().requires_grad_(), gains[1].clone().requires_grad_()
    q, k, v = parts(leaf, Hq, Hk)
    qr, kr = N.record_qk_norm_rope(q, k, gq, gk, EPS, cos, sin, halfsplit)
    o = W.record_sdpa_window(qr, kr, v, D ** -0.5, left, 0, sinks, n)
    d = torch.randn(o.shape, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    got = torch.autograd.grad(o, (leaf, gq, gk), d)
    # stage by stage
    q, k, v = parts(joint, Hq, Hk)
    q1, k1 = N.qk_norm_rope(q, k, *gains, EPS, cos, sin, halfsplit)
    rows = torch.arange(S).expand(B, S)
    for y, x, g in ((q1, q, gains[0]), (k1, k, gains[1])):
        want, size = reference(x.cpu(), g.cpu(), EPS, cos.cpu(), sin.cpu(), halfsplit, rows)
        close(y, want, F32 * size)
    fwd = W.sdpa_window_train_fwd(q1, k1, v, D ** -0.5, left, 0, sinks, n)
    ref = forward(q1, k1, v, D ** -0.5, left, 0, sinks, [S] * B if lens is None else lens, [0] * B)
    check_forward(fwd.o, fwd.stats, ref, dtype)
    assert torch.equal(o, fwd.o)
    att = W.sdpa_window_backward(fwd, d)
    check_backward((att.d_q, att.d_k, att.d_v), backward(q1, k1, v, d, D ** -0.5, ref, Hq // Hk))
    g = N.qk_norm_rope_backward(att.d_q, att.d_k, q, k, *gains, EPS, cos, sin, halfsplit)
    for x, y in zip((*parts(got[0], Hq, Hk), got[1], got[2]), (g.d_q, g.d_k, att.d_v, g.d_q_norm, g.d_k_norm)):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_a_prompt_and_single_tokens_against_a_cache():
    """Sequences of different lengths; the keys go to their rows of the cache rotated.  The single-token step is captured and replayed, the
    lengths moving on between replays; every step against float64 over what the cache then holds, and the bits of an eager step."""
    B, cap, Hq, Hk, D, left, sinks = 3, 400, 8, 2, 128, 60, 4
    prompt = [130, 64, 1]
    S = max(prompt)
    joint, gains = layer(B, S, Hq, Hk, D, BF, 3)
    cos, sin = (t.cuda() for t in tables(cap, D))
    kc, vc = (torch.full((B, cap, Hk, D), float("nan"), dtype=BF, device="cuda") for _ in range(2))
    lens = torch.tensor(prompt, dtype=torch.int32).cuda()
    q, k, v = parts(joint, Hq, Hk)
    q1, _ = N.qk_norm_rope(q, k, *gains, EPS, cos, sin, True, k_out=kc[:, :S])       # (rows of padding are written over later)
    vc[:, :S] = v
    o = W.sdpa_window(q1, kc, vc, D ** -0.5, left, 0, sinks, kv_lens=lens)
    host = lambda: [torch.nan_to_num(t.cpu()) for t in (kc, vc)]
    check_forward(o, None, forward(q1, *host(), D ** -0.5, left, 0, sinks, prompt, [0] * B), BF)
    for b in range(B):
        assert torch.isfinite(o[b]).all()

    new, (which,) = torch.empty((B, 1, Hq + 2 * Hk, D), dtype=BF, device="cuda"), (torch.arange(B).cuda(),)

    def step():
        at = lens.long()                                               # the new token's position
        q, k, v = parts(new, Hq, Hk)
        q1, k1 = N.qk_norm_rope(q, k, *gains, EPS, cos, sin, True, positions=at.view(B, 1))
        kc.index_put_((which, at), k1[:, 0])
        vc.index_put_((which, at), v[:, 0])
        return q1, W.sdpa_window_decode(q1, kc, vc, lens + 1, D ** -0.5, left, sinks)
    new.copy_(torch.randn(new.shape))
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(70):
        new.copy_(torch.randn(new.shape, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        if i % 23 == 0 or i == 69:
            n = [x + 1 for x in lens.tolist()]
            assert n == [p + i + 1 for p in prompt]
            check_forward(out[1], None, forward(out[0], *host(), D ** -0.5, left, 0, sinks, n, [x - 1 for x in n]), BF)
            got = out[1].clone()
            eager = step()
            torch.cuda.synchronize()
            assert torch.equal(got, eager[1])
        lens += 1
    # a whole prompt of the same tokens sees what the single tokens saw: the last sequence again in one call
    n = int(lens[2])
    whole = W.sdpa_window(out[0][2:], kc[2:, :n], vc[2:, :n], D ** -0.5, left, 0, sinks, q_start=n - 1)
    assert torch.equal(whole, out[1][2:])


@pytest.mark.gpu
def test_both_host_paths_give_the_same_bits(monkeypatch):
    """Calls that the native host path takes, and the same through the checks in Python."""
    B, S, Hq, Hk, D = 2, 150, 6, 2, 64
    joint, gains = layer(B, S, Hq, Hk, D, BF, 5)
    cos, sin = (t.cuda() for t in tables(S, D))
    lens, pos = torch.tensor([150, 60]).cuda(), torch.arange(S).flip(0).cuda()
    q, k, v = parts(joint, Hq, Hk)
    d = torch.randn(q.shape, device="cuda").to(BF)

    def run():
        out = list(N.qk_norm_rope(q, k, *gains, EPS, cos, sin, True, pos))
        g = N.qk_norm_rope_backward(d, d[:, :, :Hk], q, k, *gains, EPS, cos, sin, False)
        fwd = W.sdpa_window_train_fwd(q, k, v, 0.1, 40, 2, 3, lens)
        a = W.sdpa_window_backward(fwd, d)
        return out + [g.d_q, g.d_k, g.d_q_norm, g.d_k_norm, fwd.o, fwd.o_rest, fwd.stats, a.d_q, a.d_k, a.d_v,
                      W.sdpa_window(q, k, v, 0.1, 40, q_start=lens), W.sdpa_window_decode(q[:, :1], k, v, lens, 0.1, -1)]
    native = run()
    calls = []

    class Off:
        def __getattr__(self, name):
            return lambda *a: calls.append(name)
    monkeypatch.setattr(_lib, "host", lambda: Off())
    plain = run()
    assert set(calls) == {"rope", "rope_bwd", "window", "window_bwd", "window_decode"}
    for i, (x, y) in enumerate(zip(native, plain)):
        assert torch.equal(x, y), i


@pytest.mark.gpu
def test_two_threads_on_two_streams():
    shapes = [(1, 1, 3000, 8, 2, 128), (2, 500, 500, 4, 4, 64)]
    data = []
    for i, (B, Sq, Skv, Hq, Hk, D) in enumerate(shapes):
        g = torch.Generator().manual_seed(i)
        q, k, v = (torch.randn(s, generator=g).to(BF).cuda() for s in ((B, Sq, Hq, D), (B, Skv, Hk, D), (B, Skv, Hk, D)))
        lens = torch.tensor([Skv] * B).cuda()
        data.append((q, k, v, lens))

    def run(i):
        q, k, v, lens = data[i]
        if i == 0:
            return [W.sdpa_window_decode(q, k, v, lens, 0.1, -1)]
        fwd = W.sdpa_window_train_fwd(q, k, v, 0.1, 50, 0, 2)
        g = W.sdpa_window_backward(fwd, q)
        return [fwd.o, g.d_q, g.d_k, g.d_v]
    want = [run(0), run(1)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(30):
                    got = run(i)
                    s.synchronize()
                    wrong.extend(i for x, y in zip(got, want[i]) if not torch.equal(x, y))
        except Exception as e:
            wrong.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1, 0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.gpu
def test_outputs_whose_rows_coincide_are_refused():
    joint, gains = layer(2, 8, 4, 2, 64, BF)
    q, k, _ = parts(joint, 4, 2)
    for out in (torch.empty((1, 8, 2, 64), dtype=BF, device="cuda").expand(2, 8, 2, 64), torch.empty((2, 8, 1, 64), dtype=BF, device="cuda").expand(2, 8, 2, 64)):
        with pytest.raises(Error, match="lie apart"):
            N.qk_norm_rope(q, k, *gains, EPS, None, None, k_out=out)


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    joint, gains = layer(1, 20, 2, 2, 64, BF)
    leaf = joint.requires_grad_()
    q, k, v = parts(leaf, 2, 2)
    qr, kr = N.record_qk_norm_rope(q, k, *gains, EPS, None, None)
    o = W.record_sdpa_window(qr, kr, v, 0.1, 5)
    (g,) = torch.autograd.grad(o.float().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), leaf)
