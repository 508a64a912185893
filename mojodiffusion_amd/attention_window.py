"""Attention over a sliding window, with a few first tokens that stay visible: forward, training and serving forms.

The reference's attention is full (serenitymojo/ops/attention.mojo:1690-1936) or masked by an additive tensor; here the mask is a rule on
positions, and the keys it hides are not computed.  A query at position p sees key j of its sequence when

    j <= p + right   and   (j >= p - left  or  j < sinks)

left or right -1: no bound on that side (left=-1, right=0: causal attention).  Tensors are [B, S, H, Dh], BF16 or F16 (no
quantization); k and v may have fewer heads than q, which then share them in order (q's heads h*Hq/Hk .. use key head h, the
repeat_kv of models/dit/krea2_dit.mojo:703-705 without the copies).  Any strides with dense, 16-byte aligned rows.
"""
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .attention_sage import Error, SdpaFlashGrads
from .norm_rope import _rows, _rows_ok, _scratch, _strides

_TYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16}
# Calls that meet every check go through the native host path (_lib.host(), csrc/sage_torch.cpp), which returns None for the others;
# those continue below, where the checks are stated.


@dataclass
class SdpaWindowFwd:
    """What sdpa_window_train_fwd leaves for sdpa_window_backward; stats: F32 [B,H,S,1], the log-sum-exp of the visible scores; o_rest:
    what rounding to o's type left of the output (the backward's row sums are taken with it)."""
    o: torch.Tensor
    o_rest: torch.Tensor
    stats: torch.Tensor
    q: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor
    scale: float
    left: int
    right: int
    sinks: int
    kv_lens: Optional[torch.Tensor]
    q_start: int


def _check(name, q, k, v, scale, left, right, sinks):
    if q.dim() != 4 or k.dim() != 4:
        raise Error("%s: q/k/v must be rank-4 [B,S,H,Dh]" % name)
    if k.shape != v.shape:
        raise Error("%s: k/v shape mismatch" % name)
    if q.dtype not in _TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise Error("%s: q/k/v must be BF16 or F16, all the same" % name)
    if q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise Error("%s: q and k/v disagree on B/Dh" % name)
    if q.numel() == 0 or k.numel() == 0:
        raise Error("%s: empty q or k" % name)
    if q.shape[2] % k.shape[2]:
        raise Error("%s: %d query heads cannot share %d key heads" % (name, q.shape[2], k.shape[2]))
    if q.shape[3] not in (64, 128, 256):
        raise Error("%s: Dh=%d is not supported (64, 128 or 256)" % (name, q.shape[3]))
    if not 0.0 < scale < float("inf"):
        raise Error("%s: scale must be positive" % name)
    if left < -1 or right < -1 or sinks < 0:
        raise Error("%s: left and right must be at least -1, sinks at least 0" % name)


def _check_device(name, q, *others):
    for t in (q, *others):
        if t is not None and not t.is_cuda:
            raise Error("%s: tensors must live on the GPU (no CPU fallback exists)" % name)
        if t is not None and t.device != q.device:
            raise Error("%s: tensors must live on one device" % name)


def _lens(name, what, t, B):
    """int32 [B], dense."""
    if t is None:
        return None
    if t.dtype not in (torch.int32, torch.int64) or t.shape != (B,):
        raise Error("%s: %s must be int32 or int64 [B]" % (name, what))
    return t


def _int32(t):
    """t as dense int32, what lies beyond as the nearer end."""
    if t is not None and t.dtype == torch.int64:
        t = t.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)
    return None if t is None else t.contiguous()


def _start(name, q_start):
    start = int(q_start)
    if not -2 ** 29 <= start <= 2 ** 29:
        raise Error("%s: q_start=%d is not supported (at most 2^29 either way)" % (name, start))
    return start


def _ptr(t):
    return None if t is None else t.data_ptr()


def _bound(x):
    """The C argument for a number of keys: beyond any length all are alike."""
    return min(int(x), 2 ** 30)


def _forward(name, q, k, v, scale, left, right, sinks, kv_lens, q_start, training):
    r = _lib.host().window(q, k, v, scale, left, right, sinks, kv_lens, q_start, int(training))
    if r is not None:
        return (*r, q, k, v, kv_lens) if training else (r,)
    _check(name, q, k, v, scale, left, right, sinks)
    B, Sq, Hq, Dh = q.shape
    Skv, Hk = k.shape[1], k.shape[2]
    kv_lens = _lens(name, "kv_lens", kv_lens, B)
    starts = _lens(name, "q_start", q_start, B) if isinstance(q_start, torch.Tensor) else None
    start = 0 if starts is not None else _start(name, q_start)
    _check_device(name, q, k, v, kv_lens, starts)
    L = _lib.lib()
    with torch.cuda.device(q.device):
        qi, ki, vi, lens, starts = _rows(q), _rows(k), _rows(v), _int32(kv_lens), _int32(starts)
        o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        rest, stats = (torch.empty_like(o), torch.empty((B, Hq, Sq, 1), dtype=torch.float32, device=q.device)) if training else (None, None)
        ws = _scratch(L.mi355_sage_window_workspace_bytes(B, Hq, Hk, Sq, Skv, Dh, _bound(left), _bound(right), _bound(sinks)), o)
        rc = L.mi355_sage_sdpa_window(
            qi.data_ptr(), ki.data_ptr(), vi.data_ptr(), o.data_ptr(), _ptr(rest), _ptr(stats), B, Hq, Hk, Sq, Skv, Dh, _TYPES[q.dtype], float(scale),
            _strides(qi), _strides(ki), _strides(vi), _strides(o), 0, 0, 0, 0, 0, _bound(left), _bound(right), _bound(sinks), _ptr(lens), _ptr(starts),
            start, torch.cuda.current_stream(q.device).cuda_stream, ws.data_ptr(), ws.numel())
    if rc != 0:
        raise Error("%s: shim rc=%d (B=%d Sq=%d Skv=%d Hq=%d Hk=%d Dh=%d)" % (name, rc, B, Sq, Skv, Hq, Hk, Dh))
    return o, rest, stats, qi, ki, vi, lens


def sdpa_window(q, k, v, scale, left, right=0, sinks=0, kv_lens=None, q_start=0):
    """Attention of q [B,Sq,Hq,Dh] over k/v [B,Skv,Hk,Dh] through the window; returns [B,Sq,Hq,Dh] in q's type.

    kv_lens: int32 or int64 [B] on the device, the sequences' lengths (keys from there on are padding: hidden, never read); None: all
    Skv.  q_start: the position of every sequence's first query, an int or int32 / int64 [B] on the device (a
    chunk of a prompt whose first part is already in the cache), within 2^29 either way (an int beyond is refused, an element taken as the nearer end).  A query that sees no key gives zeros; one that sees some and holds a NaN or an
    infinity gives NaN in its own row."""
    return _forward("sdpa_window", q, k, v, scale, left, right, sinks, kv_lens, q_start, False)[0]


def sdpa_window_decode(q, k_cache, v_cache, kv_lens, scale, left, sinks=0):
    """The last Sq tokens of every sequence (one, or a few) against its cache [B,capacity,Hk,Dh]: query i of sequence b stands at
    kv_lens[b] - Sq + i and sees keys up to itself through the window.  kv_lens counts the keys in the cache, the new tokens'
    among them.  Queries before a sequence's first token (kv_lens[b] < Sq) give zeros."""
    o = _lib.host().window_decode(q, k_cache, v_cache, kv_lens, scale, left, sinks)
    if o is not None:
        return o
    name = "sdpa_window_decode"
    k, v = k_cache, v_cache
    _check(name, q, k, v, scale, left, 0, sinks)
    B, Sq, Hq, Dh = q.shape
    Skv, Hk = k.shape[1], k.shape[2]
    if kv_lens is None:
        raise Error("%s: kv_lens must be int32 or int64 [B]" % name)
    kv_lens = _lens(name, "kv_lens", kv_lens, B)
    _check_device(name, q, k, v, kv_lens)
    L = _lib.lib()
    with torch.cuda.device(q.device):
        qi, ki, vi, lens = _rows(q), _rows(k), _rows(v), _int32(kv_lens)
        o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        ws = _scratch(L.mi355_sage_window_workspace_bytes(B, Hq, Hk, Sq, Skv, Dh, _bound(left), 0, _bound(sinks)), o)
        rc = L.mi355_sage_sdpa_window_decode(
            qi.data_ptr(), ki.data_ptr(), vi.data_ptr(), o.data_ptr(), B, Hq, Hk, Sq, Skv, Dh, _TYPES[q.dtype], float(scale),
            _strides(qi), _strides(ki), _strides(vi), _strides(o), 0, 0, 0, 0, _bound(left), _bound(sinks), lens.data_ptr(),
            torch.cuda.current_stream(q.device).cuda_stream, ws.data_ptr(), ws.numel())
    if rc != 0:
        raise Error("%s: shim rc=%d (B=%d Sq=%d Skv=%d Hq=%d Hk=%d Dh=%d)" % (name, rc, B, Sq, Skv, Hq, Hk, Dh))
    return o


def sdpa_window_train_fwd(q, k, v, scale, left, right=0, sinks=0, kv_lens=None, q_start=0):
    """sdpa_window for a training step: the output with what the backward needs.  q_start: an int."""
    name = "sdpa_window_train_fwd"
    if isinstance(q_start, torch.Tensor):
        raise Error("%s: q_start must be an int" % name)
    o, rest, stats, q, k, v, lens = _forward(name, q, k, v, scale, left, right, sinks, kv_lens, q_start, True)
    return SdpaWindowFwd(o, rest, stats, q, k, v, float(scale), left, right, sinks, lens, int(q_start))


def sdpa_window_backward(fwd, d_out):
    """d_q [B,Sq,Hq,Dh], d_k, d_v [B,Skv,Hk,Dh] from a sdpa_window_train_fwd and the upstream gradient (Dh 64 or 128; the gradients of a
    shared key head are summed over its query heads; rows of padding, of keys that nothing sees and of queries that see nothing are zeros, whatever
    those rows of q, d_out, k and v hold)."""
    name = "sdpa_window_backward"
    r = _lib.host().window_bwd(fwd.q, fwd.k, fwd.v, fwd.o, fwd.o_rest, d_out, fwd.stats, fwd.scale, fwd.left, fwd.right, fwd.sinks, fwd.kv_lens, fwd.q_start)
    if r is not None:
        return SdpaFlashGrads(*r)
    q, k, v, o, rest, stats = fwd.q, fwd.k, fwd.v, fwd.o, fwd.o_rest, fwd.stats
    _check(name, q, k, v, fwd.scale, fwd.left, fwd.right, fwd.sinks)
    if q.shape[3] == 256:
        raise Error("%s: Dh=256 is not supported by the backward kernels (64 or 128)" % name)
    if d_out.dtype != q.dtype:
        raise Error("%s: d_out must have the type of the forward output" % name)
    if any(t.shape != q.shape or t.dtype != q.dtype for t in (o, rest, d_out)):
        raise Error("%s: o/d_out shape does not match q [B,S,H,Dh]" % name)
    B, Sq, Hq, Dh = q.shape
    Skv, Hk = k.shape[1], k.shape[2]
    if stats.dtype != torch.float32 or stats.numel() != B * Hq * Sq or not stats.is_contiguous():
        raise Error("%s: stats must be F32 [B,H,S,1]" % name)
    lens, start = _lens(name, "kv_lens", fwd.kv_lens, B), _start(name, fwd.q_start)
    _check_device(name, q, k, v, o, rest, d_out, stats, lens)
    L = _lib.lib()
    with torch.cuda.device(q.device):
        q, k, v, d, lens = _rows(q), _rows(k), _rows(v), _rows(d_out), _int32(lens)
        if not _rows_ok(o) or o.stride() != rest.stride() or rest.data_ptr() % 16:
            o, rest = o.clone(memory_format=torch.contiguous_format), rest.clone(memory_format=torch.contiguous_format)
        d_q = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        d_k, d_v = (torch.empty(k.shape, dtype=k.dtype, device=k.device) for _ in range(2))
        ws = _scratch(L.mi355_sage_window_bwd_workspace_bytes(B, Hq, Hk, Sq, Skv, Dh, _bound(fwd.left), _bound(fwd.right), _bound(fwd.sinks)), d_q)
        rc = L.mi355_sage_sdpa_window_bwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), rest.data_ptr(), d.data_ptr(), stats.data_ptr(), d_q.data_ptr(), d_k.data_ptr(), d_v.data_ptr(),
            B, Hq, Hk, Sq, Skv, Dh, _TYPES[q.dtype], fwd.scale, _strides(q), _strides(k), _strides(v), _strides(o), _strides(d), _strides(d_q),
            _strides(d_k), _strides(d_v), 0, 0, 0, 0, 0, 0, 0, 0, 0, _bound(fwd.left), _bound(fwd.right), _bound(fwd.sinks), _ptr(lens), start,
            torch.cuda.current_stream(q.device).cuda_stream, ws.data_ptr(), ws.numel())
    if rc != 0:
        raise Error("%s: shim rc=%d (B=%d Sq=%d Skv=%d Hq=%d Hk=%d Dh=%d)" % (name, rc, B, Sq, Skv, Hq, Hk, Dh))
    return SdpaFlashGrads(d_q, d_k, d_v)


class _SdpaWindowNode(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, left, right, sinks, kv_lens, q_start):
        if q.dim() == 4 and q.shape[3] == 256:
            raise Error("record_sdpa_window: Dh=256 is not supported by the backward kernels (64 or 128)")
        fwd = sdpa_window_train_fwd(q, k, v, scale, left, right, sinks, kv_lens, q_start)
        ctx.save_for_backward(fwd.o, fwd.o_rest, fwd.stats, fwd.q, fwd.k, fwd.v, fwd.kv_lens)
        ctx.window = (fwd.scale, left, right, sinks, fwd.q_start)
        return fwd.o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        o, rest, stats, q, k, v, lens = ctx.saved_tensors
        scale, left, right, sinks, q_start = ctx.window
        grads = sdpa_window_backward(SdpaWindowFwd(o, rest, stats, q, k, v, scale, left, right, sinks, lens, q_start), g.to(q.dtype))
        return grads.d_q, grads.d_k, grads.d_v, None, None, None, None, None, None


def record_sdpa_window(q, k, v, scale, left, right=0, sinks=0, kv_lens=None, q_start=0):
    """sdpa_window recorded for backpropagation, as attention_sage.record_sdpa records full attention: the result carries a node whose backward
    yields d_q, d_k, d_v."""
    return _SdpaWindowNode.apply(q, k, v, scale, left, right, sinks, kv_lens, q_start)
