"""qk_norm_rope where the caller says where to write."""
import pytest
import torch

from mojodiffusion_amd import norm_rope as N

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
