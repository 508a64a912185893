"""A paged cache of keys and values in 8 bits: appending to it, with norm and position rotation on the way, and attention over it.

The reference keeps no cache (its attention is serenitymojo/ops/attention.mojo:1690-1936, over whole tensors); this is what a served sequence of
tokens needs next to attention_window and attention_packed.  Codes are e4m3, with one power of two as a scale for each block of 32 tokens and key
head.  kv_append takes the place of norm_rope.qk_norm_rope in such a step, sdpa_paged that of attention_window.sdpa_window_decode.
"""
from dataclasses import dataclass

import torch

from . import _lib
from .attention_sage import Error
from .attention_window import _TYPES, _int32
from .norm_rope import _TYPES as _ROW_TYPES, _aligned, _scratch, _written

BLOCK = 32
# Calls that meet every check go through the native host path (_lib.host(), csrc/sage_torch.cpp), which returns None for the others;
# those continue below, where the checks are stated.


@dataclass
class KvPages:
    """The pages: codes of k [pages, blocks of a page, Hk, 32, Dh] and of v [pages, blocks of a page, Hk, Dh, 32] (a channel after the other), their scales
    [pages, blocks of a page, Hk].  A value is its code times its scale."""
    k: torch.Tensor                 # float8_e4m3fn
    v: torch.Tensor
    k_scale: torch.Tensor           # F32, powers of two
    v_scale: torch.Tensor

    @staticmethod
    def empty(pages, heads, dh, page=64, device="cuda"):
        """Pages of `page` tokens (32, 64, 128, ...) that hold nothing yet; what an append has not written is undefined."""
        if pages <= 0 or heads <= 0 or page < BLOCK or page & (page - 1) or page > 65536:
            raise Error("KvPages: pages and heads must be positive, a page 32, 64, 128, .. tokens")
        if dh not in (64, 128, 256):
            raise Error("KvPages: Dh=%d is not supported (64, 128 or 256)" % dh)
        n = page // BLOCK
        codes = lambda *s: torch.empty((pages, n, heads, *s), dtype=torch.float8_e4m3fn, device=device)
        scale = lambda: torch.ones((pages, n, heads), dtype=torch.float32, device=device)
        return KvPages(codes(BLOCK, dh), codes(dh, BLOCK), scale(), scale())

    def dense(self, page_table, length):
        """(k, v) F32 [length, Hk, Dh]: the values of one sequence's first `length` tokens, from its row of the page table.  Entries that the tokens do not need are
        not looked at; tokens whose page is not one of the cache's are NaN."""
        if page_table.dim() != 1 or not 0 <= length <= page_table.shape[0] * self.k.shape[1] * BLOCK:
            raise Error("KvPages.dense: one row of a page table that holds the tokens")
        pages = page_table[:-(-length // (self.k.shape[1] * BLOCK))].long()
        rows = pages.clamp(0, self.k.shape[0] - 1)
        values = lambda t, scale: (t.view(torch.uint8)[rows].view(t.dtype).float() * scale[rows][..., None, None]).masked_fill_((rows != pages).view(-1, 1, 1, 1, 1), torch.nan)
        k, v = values(self.k, self.k_scale), values(self.v, self.v_scale)
        flat = lambda t: t.flatten(0, 2)[:length]
        return flat(k.permute(0, 1, 3, 2, 4)), flat(v.permute(0, 1, 4, 2, 3))


def _check_cache(name, cache, page_table, kv_lens):
    """B, Hk, Dh, tokens of a page."""
    if cache.k.dim() != 5 or cache.v.dim() != 5 or cache.k_scale.dim() != 3:
        raise Error("%s: pages must be [pages, blocks, Hk, 32, Dh] and [pages, blocks, Hk, Dh, 32], scales [pages, blocks, Hk]" % name)
    P, n, Hk, block, Dh = cache.k.shape
    if block != BLOCK or cache.v.shape != (P, n, Hk, Dh, BLOCK) or cache.k_scale.shape != (P, n, Hk) or cache.v_scale.shape != (P, n, Hk):
        raise Error("%s: pages must be [pages, blocks, Hk, 32, Dh] and [pages, blocks, Hk, Dh, 32], scales [pages, blocks, Hk]" % name)
    if cache.k.dtype != torch.float8_e4m3fn or cache.v.dtype != torch.float8_e4m3fn or cache.k_scale.dtype != torch.float32 or cache.v_scale.dtype != torch.float32:
        raise Error("%s: pages must be float8_e4m3fn, scales F32" % name)
    if cache.k.numel() == 0 or n & (n - 1) or n > 2048:
        raise Error("%s: a page holds 32, 64, 128, .. tokens" % name)
    if Dh not in (64, 128, 256):
        raise Error("%s: Dh=%d is not supported (64, 128 or 256)" % (name, Dh))
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        if not t.is_contiguous() or t.data_ptr() % 16:
            raise Error("%s: pages and scales must be dense and 16-byte aligned" % name)
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.numel() == 0 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise Error("%s: page_table must be int32 [B,pages of a sequence], with dense rows" % name)
    B = page_table.shape[0]
    if kv_lens.dtype not in (torch.int32, torch.int64) or kv_lens.shape != (B,):
        raise Error("%s: kv_lens must be int32 or int64 [B]" % name)
    return B, Hk, Dh, n * BLOCK


def _same_device(name, first, *others):
    for t in (first, *others):
        if t is not None and not t.is_cuda:
            raise Error("%s: tensors must live on the GPU (no CPU fallback exists)" % name)
        if t is not None and t.device != first.device:
            raise Error("%s: tensors must live on one device" % name)


def _rows(t):
    """t [B,S,H,Dh] or [T,H,Dh], or a dense copy of it where its rows are not dense or not 16-byte aligned."""
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in t.stride()[:-1])
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _strides(t):
    """Element strides of [B,S,H,Dh] or of packed [T,H,Dh] as logical [B,H,S,Dh]."""
    s = t.stride() if t.dim() == 4 else (0, *t.stride())
    return (_lib.ctypes.c_int64 * 4)(s[0], s[2], s[1], s[3])


def _cache_args(cache, page, page_table, lens):
    return (cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), cache.k.shape[0], page, page_table.data_ptr(),
            page_table.stride(0), page_table.shape[1], lens.data_ptr())


def kv_append(cache, k, v, page_table, kv_lens, cu_seqlens=None, k_norm=None, eps=1e-6, cos=None, sin=None, halfsplit=False, q=None, q_norm=None, q_out=None):
    """Stores the last tokens of every sequence; returns q rotated (None without q).

    k, v: [B,S,Hk,Dh], the last S tokens of every sequence, or, with cu_seqlens (int32 [B+1] on the device, not falling, from 0), [T,Hk,Dh]:
    rows cu_seqlens[b] .. cu_seqlens[b+1] - 1 are sequence b's last.  BF16 or F16; any strides with dense rows, so the parts of a joint projection go in as
    they are.  page_table: int32 [B,pages of a sequence], pages of cache in the order of the tokens; kv_lens: int32 or int64 [B], lengths
    with the new tokens among them; both on the device.  Token i of a sequence's n new ones stands at kv_lens[b] - n + i.

    k's rows are divided by their root mean square (eps inside the root) times k_norm [Dh], if that is given, and rotated by the rows of cos / sin
    [rows, rot/2] that their positions name, if those are given (halfsplit and types as in norm_rope.qk_norm_rope; a position that is not in the
    tables: NaN); v's go as they are.  q [B,S,Hq,Dh] or [T,Hq,Dh] likewise, with q_norm, into a new tensor or q_out (which may be q itself and must otherwise
    overlap nothing); rows of q that belong to no sequence come out as zeros.

    A block (32 tokens of a page and head) has the least power of two as its scale with which its largest value stays within 448, at least 2^-100; while
    it fills, the scale only rises, and codes that are there are rounded again to the new one.  Values that are not finite become NaN.  Tokens before a
    sequence's first, beyond its pages, or whose page is not one of cache's are not stored.  Pages that sequences share must be full ones; every other is one sequence's own."""
    r = _lib.host().kv_append(cache.k, cache.v, cache.k_scale, cache.v_scale, k, v, page_table, kv_lens, cu_seqlens, k_norm, eps, cos, sin, halfsplit, q, q_norm) \
        if q_out is None else None
    if r is not None:
        return None if q is None else r
    name = "kv_append"
    B, Hk, Dh, page = _check_cache(name, cache, page_table, kv_lens)
    packed = cu_seqlens is not None
    if packed and (cu_seqlens.dtype not in (torch.int32, torch.int64) or cu_seqlens.shape != (B + 1,)):
        raise Error("%s: cu_seqlens must be int32 or int64 [B+1]" % name)
    for t in (k, v):
        if t.dim() != (3 if packed else 4) or t.shape[-2:] != (Hk, Dh) or (not packed and t.shape[0] != B) or t.shape != k.shape:
            raise Error("%s: k/v must be [B,S,Hk,Dh], or [T,Hk,Dh] with cu_seqlens, both the same" % name)
        if t.dtype not in _TYPES or t.dtype != k.dtype:
            raise Error("%s: k/v must be BF16 or F16, both the same" % name)
    if q is not None and (q.dim() != k.dim() or q.shape[:-2] != k.shape[:-2] or q.shape[-1] != Dh or q.dtype != k.dtype or q.numel() == 0):
        raise Error("%s: q must be [B,S,Hq,Dh] or [T,Hq,Dh], of k's type" % name)
    if q is None and (q_out is not None or q_norm is not None):
        raise Error("%s: q_norm or q_out without q" % name)
    if k.numel() == 0:
        raise Error("%s: empty k" % name)
    if not eps >= 0.0:
        raise Error("%s: eps must not be negative" % name)
    gains = [g for g in (q_norm, k_norm) if g is not None]
    for g in gains:
        if g.dim() != 1 or g.numel() != Dh:
            raise Error("%s: weight must be [%d]" % (name, Dh))
        if g.dtype not in _ROW_TYPES or g.dtype != gains[0].dtype:
            raise Error("%s: weights must be BF16, F16 or F32, both the same" % name)
    if (cos is None) != (sin is None):
        raise Error("%s: cos and sin come together" % name)
    rot = 0
    if cos is not None:
        if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[0] == 0:
            raise Error("%s: cos/sin must be [rows, rot/2]" % name)
        if cos.dtype != sin.dtype or cos.dtype not in _ROW_TYPES:
            raise Error("%s: cos/sin tables must be BF16, F16 or F32, both the same" % name)
        rot = 2 * cos.shape[1]
        if rot > Dh or rot % 16 or rot == 0:
            raise Error("%s: %d rotated channels are not supported (a multiple of 16 up to Dh=%d)" % (name, rot, Dh))
    if q_out is not None:
        if q_out.shape != q.shape or q_out.dtype != q.dtype:
            raise Error("%s: an output must have the shape, type and device of its input" % name)
        if q_out.stride(-1) != 1 or q_out.data_ptr() % 16 or any(s % 8 for s in q_out.stride()[:-1]):
            raise Error("%s: rows of an output must be dense and 16-byte aligned" % name)
        if any(n > 1 and s == 0 for n, s in zip(q_out.shape, q_out.stride())):
            raise Error("%s: rows of an output must lie apart" % name)
    _same_device(name, k, v, q, q_out, cache.k, cache.v, cache.k_scale, cache.v_scale, page_table, kv_lens, cu_seqlens, k_norm, q_norm, cos, sin)
    with torch.cuda.device(k.device):
        ki, vi, qi, lens, cu = _rows(k), _rows(v), None if q is None else _rows(q), _int32(kv_lens), _int32(cu_seqlens)
        qo = None if q is None else torch.empty(q.shape, dtype=q.dtype, device=q.device) if q_out is None else q_out
        gq, gk = (None if g is None else _aligned(g) for g in (q_norm, k_norm))
        table = (None, None, 0, 0, 0, 0)
        if rot:
            esz = cos.element_size()
            if not all(t.stride(1) == 1 and t.data_ptr() % 16 == 0 and t.stride(0) * esz % 16 == 0 for t in (cos, sin)) or cos.stride(0) != sin.stride(0):
                cos, sin = _aligned(cos), _aligned(sin)
            table = (cos.data_ptr(), sin.data_ptr(), _ROW_TYPES[cos.dtype], rot, cos.shape[0], cos.stride(0))
        ptr = lambda t: None if t is None else t.data_ptr()
        rc = _lib.lib().mi355_sage_kv_append(
            ki.data_ptr(), vi.data_ptr(), ptr(qi), ptr(qo), *_cache_args(cache, page, page_table, lens), ptr(cu), B, k.shape[0] if packed else k.shape[1],
            0 if q is None else q.shape[-2], Hk, Dh, _TYPES[k.dtype], _strides(ki), _strides(vi), None if q is None else _strides(qi), None if q is None else _strides(qo),
            0, 0, 0, 0, ptr(gq), ptr(gk), _ROW_TYPES[gains[0].dtype] if gains else 0, float(eps), *table, int(halfsplit), torch.cuda.current_stream(k.device).cuda_stream)
    if rc != 0:
        raise Error("%s: shim rc=%d (B=%d rows=%d Hk=%d Dh=%d)" % (name, rc, B, k.numel() // (Hk * Dh), Hk, Dh))
    _written(cache.k, cache.v, cache.k_scale, cache.v_scale, q_out)
    return qo


def sdpa_paged(q, cache, page_table, kv_lens, scale):
    """The last Sq tokens of every sequence (one, or a few) against the cache: q [B,Sq,Hq,Dh], BF16 or F16 -> [B,Sq,Hq,Dh].

    Query i of sequence b stands at kv_lens[b] - Sq + i and sees keys up to itself; kv_lens counts the keys in the cache, the new tokens' among them.  Queries
    before a sequence's first token (kv_lens[b] < Sq) give zeros; a length beyond its row of the page table counts as what that holds.  q's heads h*Hq/Hk .. share key head h.  page_table and kv_lens as in kv_append; a
    sequence one of whose pages is not one of cache's gives NaN."""
    o = _lib.host().paged(q, cache.k, cache.v, cache.k_scale, cache.v_scale, page_table, kv_lens, scale)
    if o is not None:
        return o
    name = "sdpa_paged"
    B, Hk, Dh, page = _check_cache(name, cache, page_table, kv_lens)
    if q.dim() != 4 or q.shape[0] != B or q.shape[3] != Dh or q.numel() == 0:
        raise Error("%s: q must be [B,Sq,Hq,Dh] with the cache's Dh" % name)
    if q.dtype not in _TYPES:
        raise Error("%s: q must be BF16 or F16" % name)
    Sq, Hq = q.shape[1], q.shape[2]
    if Hq % Hk:
        raise Error("%s: %d query heads cannot share %d key heads" % (name, Hq, Hk))
    if not 0.0 < scale < float("inf"):
        raise Error("%s: scale must be positive" % name)
    _same_device(name, q, cache.k, cache.v, cache.k_scale, cache.v_scale, page_table, kv_lens)
    L = _lib.lib()
    with torch.cuda.device(q.device):
        qi, lens = _rows(q), _int32(kv_lens)
        o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        ws = _scratch(L.mi355_sage_paged_workspace_bytes(B, Hq, Hk, Sq, Dh, page_table.shape[1], page), o)
        rc = L.mi355_sage_sdpa_paged(
            qi.data_ptr(), o.data_ptr(), *_cache_args(cache, page, page_table, lens), B, Hq, Hk, Sq, Dh, _TYPES[q.dtype], float(scale), _strides(qi), _strides(o), 0, 0,
            torch.cuda.current_stream(q.device).cuda_stream, ws.data_ptr(), ws.numel())
    if rc != 0:
        raise Error("%s: shim rc=%d (B=%d Sq=%d Hq=%d Hk=%d Dh=%d)" % (name, rc, B, Sq, Hq, Hk, Dh))
    return o
