"""qk_norm_rope where the caller says where to write."""
import ctypes

import pytest
import torch

from mojodiffusion_amd import _lib
from mojodiffusion_amd import norm_rope as N
from mojodiffusion_amd.attention_sage import Error

BF = torch.bfloat16


def projections(B=2, S=9, Hq=4, Hk=2, D=64):
    g = torch.Generator().manual_seed(0)
    return [torch.randn(s, generator=g).to(BF).cuda() for s in ((B, S, Hq, D), (B, S, Hk, D))] + [(1 + 0.3 * torch.randn(D, generator=g)).cuda() for _ in range(2)]


@pytest.mark.gpu
def test_torch_knows_what_was_written():
    """A tensor that a node has saved and a call writes over: torch's error in the backward, not a wrong gradient."""
    q, k, gq, gk = projections()
    for which in ("q_out", "k_out"):
        x = (q if which == "q_out" else k).clone()
        w = torch.ones_like(x, requires_grad=True)
        y = (w * x).sum()                                              # (saves x)
        before = x._version
        N.qk_norm_rope(q, k, gq, gk, 1e-6, None, None, **{which: x})
        assert x._version == before + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    # rows of a cache: its views share the count
    cache = torch.zeros((2, 20, 2, 64), dtype=BF, device="cuda")
    N.qk_norm_rope(q, k, gq, gk, 1e-6, None, None, k_out=cache[:, 5:14])
    assert cache._version == 1
    with torch.inference_mode():
        cache = torch.zeros((2, 20, 2, 64), dtype=BF, device="cuda")
    N.qk_norm_rope(q, k, gq, gk, 1e-6, None, None, k_out=cache[:, 5:14])        # (an inference tensor has none)
    assert torch.equal(cache[:, 5:14], N.qk_norm_rope(q, k, gq, gk, 1e-6, None, None)[1])


def test_outputs_over_the_other_input_are_refused():
    """Q's rows written over K's, which another workgroup has still to read, or the other way; both outputs in one place; an input's own place with
    other strides.  (Codes only: the addresses are made up and not read.)"""
    L = _lib.lib()
    A = 1 << 20
    st, other = _lib.strides_bhnd(8, 4, 64), (ctypes.c_int64 * 4)(4 * 8 * 64, 8 * 64, 64, 1)

    def call(q=A, k=2 * A, qo=3 * A, ko=4 * A, qs=st, qos=st, kos=st, off=(0, 0, 0, 0)):
        return L.mi355_sage_qk_norm_rope(q, k, qo, ko, 1, 8, 4, 4, 64, 0, qs, st, qos, kos, *off, A, A, 2, 1e-6, None, None, 0, 0, 0, 0, 0, None, 0, 0, None)

    for change in (dict(qo=2 * A), dict(ko=A), dict(qo=2 * A, ko=A), dict(ko=3 * A), dict(qo=A, qos=other), dict(ko=2 * A, kos=other), dict(qo=A, off=(0, 0, A // 2, 0))):
        assert call(**change) == -1, change

    def back(dqo=A, dko=2 * A, q=3 * A, k=4 * A, dq=5 * A, dk=6 * A, dqs=st, room=1 << 20):
        return L.mi355_sage_qk_norm_rope_bwd(dqo, dko, q, k, dq, dk, A, A, 1, 8, 4, 4, 64, 0, st, st, st, st, dqs, st, 0, 0, 0, 0, 0, 0, A, A, 2, 1e-6, None, None, 0, 0, 0,
                                             0, 0, None, 0, 0, None, A, room)

    for change in (dict(dq=2 * A), dict(dk=A), dict(dq=4 * A), dict(dk=3 * A), dict(dk=5 * A), dict(dq=A, dqs=other)):
        assert back(**change) == -1, change
    assert back(dq=A, dk=2 * A, room=8) == -3                                  # (in place: allowed, stopped by its workspace)


@pytest.mark.gpu
def test_outputs_over_the_other_input_are_refused_on_the_device():
    q, k, gq, gk = projections(Hq=2, Hk=2)
    before = [t.clone() for t in (q, k)]
    for outs in (dict(q_out=k), dict(k_out=q), dict(q_out=k, k_out=q)):
        with pytest.raises(Error, match="rc=-1"):
            N.qk_norm_rope(q, k, gq, gk, 1e-6, None, None, **outs)
    assert all(torch.equal(x, y) for x, y in zip((q, k), before)) and q._version == k._version == 0
    want = N.qk_norm_rope(q, k, gq, gk, 1e-6, None, None)
    N.qk_norm_rope(q, k, gq, gk, 1e-6, None, None, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
