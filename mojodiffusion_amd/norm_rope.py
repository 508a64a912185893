"""RMSNorm of every query and key head and the position rotation, as an operator with its gradient.

The reference calls rms_norm (serenitymojo/ops/norm.mojo:152) and rope_interleaved / rope_halfsplit
(serenitymojo/ops/rope.mojo:373, :10-13) on Q and on K, e.g. serenitymojo/models/klein/single_block.mojo:977-981.
attention_sage.qk_norm_rope_sdpa_nomask fuses the same steps into the quantizers of full attention; the calls here
leave the normalised, rotated rows themselves, for attention that takes them (attention_window, a cache, the
backward of either), with fp32 arithmetic between the rows read and the rows written, and give the gradients
of the projections and of both gains.

Tensors are [B, S, H, Dh]; any strides with dense, 16-byte aligned rows, so the parts of a joint projection go in as they are.
"""
from dataclasses import dataclass

import torch

from . import _lib
from .attention_sage import Error

# Calls that meet every check go through the native host path (_lib.host(), csrc/sage_torch.cpp), which returns None for the others;
# those continue below, where the checks are stated.
_TYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16, torch.float32: _lib.F32}


@dataclass
class QkNormRopeGrads:
    d_q: torch.Tensor
    d_k: torch.Tensor
    d_q_norm: torch.Tensor          # F32 [Dh]
    d_k_norm: torch.Tensor


def _scratch(nbytes, like):
    """A workspace of a call's own, from torch's allocator: calls on other streams and captured graphs (whose pool it comes from
    under capture) never share it."""
    return torch.empty(max(nbytes, 256), dtype=torch.uint8, device=like.device)


def _rows_ok(t):
    per = 16 // t.element_size()
    return t.stride(3) == 1 and t.data_ptr() % 16 == 0 and all(s % per == 0 for s in t.stride()[:3])


def _rows(t):
    """t, or a dense copy of it where its rows are not dense or not 16-byte aligned."""
    return t if _rows_ok(t) else t.clone(memory_format=torch.contiguous_format)


def _strides(t):
    """Element strides of a [B,S,H,Dh] tensor as logical [B,H,S,Dh]."""
    s = t.stride()
    return (_lib.ctypes.c_int64 * 4)(s[0], s[2], s[1], s[3])


def _aligned(t):
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _check(name, q, k, q_norm, k_norm, eps, cos, sin, positions):
    """Checks of both directions; returns the trailing arguments of the C calls and what they point to."""
    if q.dim() != 4 or k.dim() != 4:
        raise Error("%s: q/k must be rank-4 [B,S,H,Dh]" % name)
    if q.dtype != k.dtype or q.dtype not in _TYPES:
        raise Error("%s: q/k must be BF16, F16 or F32, both the same" % name)
    if q.shape[0] != k.shape[0] or q.shape[1] != k.shape[1] or q.shape[3] != k.shape[3]:
        raise Error("%s: q and k disagree on B/S/Dh" % name)
    B, S, Hq, Dh = q.shape
    if B * S * Hq * k.shape[2] == 0:
        raise Error("%s: empty q or k" % name)
    if Dh == 0 or Dh % 16 or Dh > 256:
        raise Error("%s: Dh=%d is not supported (a multiple of 16 up to 256)" % (name, Dh))
    if not eps >= 0.0:
        raise Error("%s: eps must not be negative" % name)
    for g in (q_norm, k_norm):
        if g.dim() != 1 or g.numel() != Dh:
            raise Error("%s: weight must be [%d]" % (name, Dh))
        if g.dtype not in _TYPES or g.dtype != q_norm.dtype:
            raise Error("%s: weights must be BF16, F16 or F32, both the same" % name)
    if (cos is None) != (sin is None):
        raise Error("%s: cos and sin come together" % name)
    rot = 0
    if cos is not None:
        if cos.dim() != 2 or cos.shape != sin.shape:
            raise Error("%s: cos/sin must be [rows, rot/2]" % name)
        if cos.dtype != sin.dtype or cos.dtype not in _TYPES:
            raise Error("%s: cos/sin tables must be BF16, F16 or F32, both the same" % name)
        rot = 2 * cos.shape[1]
        if rot > Dh or rot % 16 or rot == 0:
            raise Error("%s: %d rotated channels are not supported (a multiple of 16 up to Dh=%d)" % (name, rot, Dh))
        if cos.shape[0] == 0 or (positions is None and cos.shape[0] < S):
            raise Error("%s: cos/sin hold %d rows for %d positions" % (name, cos.shape[0], S))
    if positions is not None:
        if cos is None:
            raise Error("%s: positions without tables" % name)
        if positions.dtype not in (torch.int32, torch.int64) or positions.shape not in ((B, S), (S,), (1, S)):
            raise Error("%s: positions must be int32 or int64 [B,S] or [S]" % name)
    for t in (q, k, q_norm, k_norm, cos, sin, positions):
        if t is not None and not t.is_cuda:
            raise Error("%s: tensors must live on the GPU (no CPU fallback exists)" % name)
        if t is not None and t.device != q.device:
            raise Error("%s: tensors must live on one device" % name)
    gq, gk = _aligned(q_norm), _aligned(k_norm)
    keep = [gq, gk]
    table = (None, None, 0, 0, 0, 0)
    if rot:
        esz = cos.element_size()
        if not all(t.stride(1) == 1 and t.data_ptr() % 16 == 0 and t.stride(0) * esz % 16 == 0 for t in (cos, sin)) or cos.stride(0) != sin.stride(0):
            cos, sin = _aligned(cos), _aligned(sin)
        keep += [cos, sin]
        table = (cos.data_ptr(), sin.data_ptr(), _TYPES[cos.dtype], rot, cos.shape[0], cos.stride(0))
    pos = (None, 0, 0)
    if positions is not None:
        if positions.stride(-1) != 1:
            positions = positions.contiguous()
        keep.append(positions)
        shared = positions.dim() == 1 or positions.shape[0] == 1
        pos = (positions.data_ptr(), 0 if shared else positions.stride(0), positions.element_size())
    return gq, gk, table, pos, keep


def _out(name, out, like):
    if out is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise Error("%s: an output must have the shape, type and device of its input" % name)
    if not _rows_ok(out):
        raise Error("%s: rows of an output must be dense and 16-byte aligned" % name)
    if any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
        raise Error("%s: rows of an output must lie apart" % name)
    return out


def _written(*outs):
    """Counts a write into tensors that the caller gave, as torch's own calls do: a node that has saved one of them then refuses its backward."""
    torch.autograd.graph.increment_version([t for t in outs if t is not None and not t.is_inference()])


def qk_norm_rope(q, k, q_norm, k_norm, eps, cos, sin, halfsplit=False, positions=None, q_out=None, k_out=None):
    """(q_rot, k_rot) for q [B,S,Hq,Dh] and k [B,S,Hk,Dh] of one type (BF16, F16 or F32): every head's row
    divided by its root mean square (eps inside the root), times its gain [Dh], then its first rot channels rotated by the
    token's angles.

    cos/sin: [rows, rot/2], BF16, F16 or F32, shared by the heads (the reference's tables of S*H rows,
    sampling/klein_sampler.mojo:305-307, repeat every row H times: pass cos[::H]); None for the norm alone.  rot may be less than
    Dh: the other channels pass.  halfsplit: pairs (i, i + rot/2) instead of (2i, 2i+1).  positions: int32 or int64
    [B,S] or [S], rows of the tables by token (a token whose position is not in the tables comes out as NaN);
    without it token s takes row s.  q_out/k_out: where to write, e.g. rows of a cache; q_out may be q itself and k_out k; otherwise
    they must overlap neither q, k nor each other."""
    if q_out is None and k_out is None:
        r = _lib.host().rope(q, k, q_norm, k_norm, eps, cos, sin, halfsplit, positions)
        if r is not None:
            return r
    name = "qk_norm_rope"
    gq, gk, table, pos, keep = _check(name, q, k, q_norm, k_norm, eps, cos, sin, positions)
    B, S, Hq, Dh = q.shape
    qi, ki = _rows(q), _rows(k)
    qo, ko = _out(name, q_out, q), _out(name, k_out, k)
    with torch.cuda.device(q.device):
        rc = _lib.lib().mi355_sage_qk_norm_rope(
            qi.data_ptr(), ki.data_ptr(), qo.data_ptr(), ko.data_ptr(), B, S, Hq, k.shape[2], Dh, _TYPES[q.dtype],
            _strides(qi), _strides(ki), _strides(qo), _strides(ko), 0, 0, 0, 0,
            gq.data_ptr(), gk.data_ptr(), _TYPES[gq.dtype], float(eps), *table, int(halfsplit), *pos,
            torch.cuda.current_stream(q.device).cuda_stream)
    if rc != 0:
        raise Error("%s: shim rc=%d (B=%d S=%d Hq=%d Hk=%d Dh=%d)" % (name, rc, B, S, Hq, k.shape[2], Dh))
    _written(q_out, k_out)
    return qo, ko


def qk_norm_rope_backward(d_q_rot, d_k_rot, q, k, q_norm, k_norm, eps, cos, sin, halfsplit=False, positions=None):
    """Gradients of qk_norm_rope from the upstream gradients of its two results and the inputs it was called with: d_q and d_k in
    q's type, the gains' in F32 (sums over every token and head; the same bits on every call)."""
    r = _lib.host().rope_bwd(d_q_rot, d_k_rot, q, k, q_norm, k_norm, eps, cos, sin, halfsplit, positions)
    if r is not None:
        return QkNormRopeGrads(*r)
    name = "qk_norm_rope_backward"
    gq, gk, table, pos, keep = _check(name, q, k, q_norm, k_norm, eps, cos, sin, positions)
    for d, x in ((d_q_rot, q), (d_k_rot, k)):
        if d.shape != x.shape or d.dtype != x.dtype or d.device != x.device:
            raise Error("%s: upstream gradients must have the shape, type and device of q and k" % name)
    B, S, Hq, Dh = q.shape
    Hk = k.shape[2]
    L = _lib.lib()
    qi, ki, dqi, dki = _rows(q), _rows(k), _rows(d_q_rot), _rows(d_k_rot)
    dq, dk = _out(name, None, q), _out(name, None, k)
    d_gain = torch.empty((2, Dh), dtype=torch.float32, device=q.device)
    with torch.cuda.device(q.device):
        ws = _scratch(L.mi355_sage_qk_norm_rope_bwd_workspace_bytes(B, S, Hq, Hk, Dh), dq)
        rc = L.mi355_sage_qk_norm_rope_bwd(
            dqi.data_ptr(), dki.data_ptr(), qi.data_ptr(), ki.data_ptr(), dq.data_ptr(), dk.data_ptr(), d_gain[0].data_ptr(),
            d_gain[1].data_ptr(), B, S, Hq, Hk, Dh, _TYPES[q.dtype], _strides(dqi), _strides(dki), _strides(qi), _strides(ki),
            _strides(dq), _strides(dk), 0, 0, 0, 0, 0, 0, gq.data_ptr(), gk.data_ptr(), _TYPES[gq.dtype], float(eps), *table,
            int(halfsplit), *pos, torch.cuda.current_stream(q.device).cuda_stream, ws.data_ptr(), ws.numel())
    if rc != 0:
        raise Error("%s: shim rc=%d (B=%d S=%d Hq=%d Hk=%d Dh=%d)" % (name, rc, B, S, Hq, Hk, Dh))
    return QkNormRopeGrads(dq, dk, d_gain[0], d_gain[1])


class _QkNormRopeNode(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_norm, k_norm, eps, cos, sin, halfsplit, positions):
        qo, ko = qk_norm_rope(q, k, q_norm, k_norm, eps, cos, sin, halfsplit, positions)
        ctx.save_for_backward(q, k, q_norm, k_norm, cos, sin, positions)
        ctx.eps, ctx.halfsplit = float(eps), bool(halfsplit)
        return qo, ko

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_q, g_k):
        q, k, q_norm, k_norm, cos, sin, positions = ctx.saved_tensors
        g = qk_norm_rope_backward(g_q.to(q.dtype), g_k.to(k.dtype), q, k, q_norm, k_norm, ctx.eps, cos, sin, ctx.halfsplit, positions)
        return g.d_q, g.d_k, g.d_q_norm.to(q_norm.dtype), g.d_k_norm.to(k_norm.dtype), None, None, None, None, None


def record_qk_norm_rope(q, k, q_norm, k_norm, eps, cos, sin, halfsplit=False, positions=None):
    """qk_norm_rope recorded for backpropagation, as attention_sage.record_sdpa records attention: the results carry a node
    whose backward yields the gradients of q, k and both gains."""
    return _QkNormRopeNode.apply(q, k, q_norm, k_norm, eps, cos, sin, halfsplit, positions)
