"""Attention over whole sequences of different lengths that lie one behind the other in one tensor, without padding: forward and training forms.

The reference pads a batch to one length and masks what is added (serenitymojo/ops/attention.mojo:1790); here a batch is [T, H, Dh], all sequences' rows,
with cu_seqlens [B+1] on the device: rows cu_seqlens[b] .. cu_seqlens[b+1] - 1 are sequence b's.  BF16 or F16 (no quantization); k and v may have fewer heads
than q, which then share them in order.  Any strides with dense, 16-byte aligned rows.  For single tokens against what a sequence has so far see
attention_window.sdpa_window_decode (a dense cache) and kv_cache.sdpa_paged.
"""
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .attention_sage import Error, SdpaFlashGrads
from .attention_window import _TYPES, _check_device, _int32
from .kv_cache import _rows, _strides
from .norm_rope import _scratch

# Calls that meet every check go through the native host path (_lib.host(), csrc/sage_torch.cpp), which returns None for the others;
# those continue below, where the checks are stated.


@dataclass
class SdpaPackedFwd:
    """What sdpa_packed_train_fwd leaves for sdpa_packed_backward; stats: F32 [Hq,T], the log-sum-exp of the visible scores; o_rest: what rounding to o's type left
    of the output."""
    o: torch.Tensor
    o_rest: torch.Tensor
    stats: torch.Tensor
    q: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor
    cu_seqlens: torch.Tensor
    cu_seqlens_k: Optional[torch.Tensor]
    scale: float
    causal: bool


def _check(name, q, k, v, cu, cu_k, scale):
    if q.dim() != 3 or k.dim() != 3:
        raise Error("%s: q/k/v must be rank-3 [T,H,Dh]" % name)
    if k.shape != v.shape:
        raise Error("%s: k/v shape mismatch" % name)
    if q.dtype not in _TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise Error("%s: q/k/v must be BF16 or F16, all the same" % name)
    if q.shape[2] != k.shape[2] or (cu_k is None and q.shape[0] != k.shape[0]):
        raise Error("%s: q and k/v disagree on T/Dh" % name)
    if q.numel() == 0 or k.numel() == 0:
        raise Error("%s: empty q or k" % name)
    if q.shape[1] % k.shape[1]:
        raise Error("%s: %d query heads cannot share %d key heads" % (name, q.shape[1], k.shape[1]))
    if q.shape[2] not in (64, 128, 256):
        raise Error("%s: Dh=%d is not supported (64, 128 or 256)" % (name, q.shape[2]))
    if not 0.0 < scale < float("inf"):
        raise Error("%s: scale must be positive" % name)
    for t in (cu, cu_k):
        if t is not None and (t.dtype not in (torch.int32, torch.int64) or t.dim() != 1 or t.numel() < 2 or t.shape != cu.shape):
            raise Error("%s: cu_seqlens must be int32 or int64 [B+1]" % name)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _forward(name, q, k, v, cu, cu_k, scale, causal, training):
    r = _lib.host().packed(q, k, v, cu, cu_k, scale, causal, int(training))
    if r is not None:
        return (*r, q, k, v, cu, cu_k) if training else (r,)
    _check(name, q, k, v, cu, cu_k, scale)
    _check_device(name, q, k, v, cu, cu_k)
    T, Hq, Dh = q.shape
    with torch.cuda.device(q.device):
        qi, ki, vi, cu, cu_k = _rows(q), _rows(k), _rows(v), _int32(cu), _int32(cu_k)
        o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        rest, stats = (torch.empty_like(o), torch.empty((Hq, T), dtype=torch.float32, device=q.device)) if training else (None, None)
        rc = _lib.lib().mi355_sage_sdpa_packed(
            qi.data_ptr(), ki.data_ptr(), vi.data_ptr(), o.data_ptr(), _ptr(rest), _ptr(stats), cu.data_ptr(), (cu if cu_k is None else cu_k).data_ptr(), cu.numel() - 1, Hq,
            k.shape[1], T, k.shape[0], Dh, _TYPES[q.dtype], float(scale), _strides(qi), _strides(ki), _strides(vi), _strides(o), 0, 0, 0, 0, 0, int(causal),
            torch.cuda.current_stream(q.device).cuda_stream)
    if rc != 0:
        raise Error("%s: shim rc=%d (B=%d T=%d Hq=%d Hk=%d Dh=%d)" % (name, rc, cu.numel() - 1, T, Hq, k.shape[1], Dh))
    return o, rest, stats, qi, ki, vi, cu, cu_k


def sdpa_packed(q, k, v, cu_seqlens, scale, causal=True, cu_seqlens_k=None):
    """Attention of every sequence's queries over its own keys: q [T,Hq,Dh], k/v [T,Hk,Dh] -> [T,Hq,Dh] in q's type.

    cu_seqlens: int32 or int64 [B+1] on the device, from 0, not falling; sequences may be empty, and rows behind the last give zeros.  causal: a query sees the keys up
    to itself, else all of its sequence.  cu_seqlens_k: the keys' own offsets, where k and v [Tk,Hk,Dh] hold more (or fewer) rows a
    sequence than q: its queries then stand at the last positions of its keys (a chunk of a prompt over all of it so far); a query before the first key
    sees none if causal and gives zeros."""
    return _forward("sdpa_packed", q, k, v, cu_seqlens, cu_seqlens_k, scale, causal, False)[0]


def sdpa_packed_train_fwd(q, k, v, cu_seqlens, scale, causal=True, cu_seqlens_k=None):
    """sdpa_packed for a training step: the output with what the backward needs (Dh 64 or 128; at 256 the statistics are what is had of it, no backward takes it)."""
    o, rest, stats, q, k, v, cu, cu_k = _forward("sdpa_packed_train_fwd", q, k, v, cu_seqlens, cu_seqlens_k, scale, causal, True)
    return SdpaPackedFwd(o, rest, stats, q, k, v, cu, cu_k, float(scale), bool(causal))


def sdpa_packed_backward(fwd, d_out):
    """d_q [T,Hq,Dh], d_k, d_v [Tk,Hk,Dh] from a sdpa_packed_train_fwd and the upstream gradient (Dh 64 or 128; the gradients of a shared key head are summed over
    its query heads; rows of queries that see no key, of keys that no query sees and behind the last sequence are zeros)."""
    name = "sdpa_packed_backward"
    r = _lib.host().packed_bwd(fwd.q, fwd.k, fwd.v, fwd.o, fwd.o_rest, d_out, fwd.stats, fwd.cu_seqlens, fwd.cu_seqlens_k, fwd.scale, fwd.causal)
    if r is not None:
        return SdpaFlashGrads(*r)
    q, k, v, o, rest, stats, cu, cu_k = fwd.q, fwd.k, fwd.v, fwd.o, fwd.o_rest, fwd.stats, fwd.cu_seqlens, fwd.cu_seqlens_k
    _check(name, q, k, v, cu, cu_k, fwd.scale)
    if q.shape[2] == 256:
        raise Error("%s: Dh=256 is not supported by the backward kernels (64 or 128)" % name)
    if d_out.dtype != q.dtype:
        raise Error("%s: d_out must have the type of the forward output" % name)
    if any(t.shape != q.shape or t.dtype != q.dtype for t in (o, rest, d_out)):
        raise Error("%s: o/d_out shape does not match q [T,H,Dh]" % name)
    T, Hq, Dh = q.shape
    Tk, Hk = k.shape[:2]
    if stats.dtype != torch.float32 or stats.numel() != Hq * T or not stats.is_contiguous():
        raise Error("%s: stats must be F32 [H,T]" % name)
    _check_device(name, q, k, v, o, rest, d_out, stats, cu, cu_k)
    L = _lib.lib()
    with torch.cuda.device(q.device):
        q, k, v, d, cu, cu_k = _rows(q), _rows(k), _rows(v), _rows(d_out), _int32(cu), _int32(cu_k)
        if _rows(o) is not o or o.stride() != rest.stride() or rest.data_ptr() % 16:
            o, rest = o.clone(memory_format=torch.contiguous_format), rest.clone(memory_format=torch.contiguous_format)
        d_q = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        d_k, d_v = (torch.empty(k.shape, dtype=k.dtype, device=k.device) for _ in range(2))
        B = cu.numel() - 1
        ws = _scratch(L.mi355_sage_packed_bwd_workspace_bytes(B, Hq, Hk, T, Tk, Dh), d_q)
        rc = L.mi355_sage_sdpa_packed_bwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), rest.data_ptr(), d.data_ptr(), stats.data_ptr(), d_q.data_ptr(), d_k.data_ptr(), d_v.data_ptr(),
            cu.data_ptr(), (cu if cu_k is None else cu_k).data_ptr(), B, Hq, Hk, T, Tk, Dh, _TYPES[q.dtype], fwd.scale, _strides(q), _strides(k), _strides(v), _strides(o),
            _strides(d), _strides(d_q), _strides(d_k), _strides(d_v), 0, 0, 0, 0, 0, 0, 0, 0, 0, int(fwd.causal), torch.cuda.current_stream(q.device).cuda_stream, ws.data_ptr(),
            ws.numel())
    if rc != 0:
        raise Error("%s: shim rc=%d (B=%d T=%d Hq=%d Hk=%d Dh=%d)" % (name, rc, B, T, Hq, Hk, Dh))
    return SdpaFlashGrads(d_q, d_k, d_v)


class _SdpaPackedNode(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, scale, causal, cu_seqlens_k):
        if q.dim() == 3 and q.shape[2] == 256:
            raise Error("record_sdpa_packed: Dh=256 is not supported by the backward kernels (64 or 128)")
        fwd = sdpa_packed_train_fwd(q, k, v, cu_seqlens, scale, causal, cu_seqlens_k)
        ctx.save_for_backward(fwd.o, fwd.o_rest, fwd.stats, fwd.q, fwd.k, fwd.v, fwd.cu_seqlens, fwd.cu_seqlens_k)
        ctx.packed = (fwd.scale, fwd.causal)
        return fwd.o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        grads = sdpa_packed_backward(SdpaPackedFwd(*ctx.saved_tensors, *ctx.packed), g.to(ctx.saved_tensors[3].dtype))
        return grads.d_q, grads.d_k, grads.d_v, None, None, None, None


def record_sdpa_packed(q, k, v, cu_seqlens, scale, causal=True, cu_seqlens_k=None):
    """sdpa_packed recorded for backpropagation, as attention_sage.record_sdpa records full attention: the result carries a node whose backward yields d_q,
    d_k, d_v."""
    return _SdpaPackedNode.apply(q, k, v, cu_seqlens, scale, causal, cu_seqlens_k)
