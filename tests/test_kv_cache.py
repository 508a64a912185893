"""Refusals of the paged cache's calls that need no device, and its sizes."""
import ctypes
import os
import subprocess

import pytest
import torch

from mojodiffusion_amd import _lib
from mojodiffusion_amd import kv_cache as C
from mojodiffusion_amd.attention_sage import Error

BF = torch.bfloat16
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mojodiffusion_amd", "csrc")


def setup(Hk=2, D=64, page=32, B=2):
    cache = C.KvPages.empty(4, Hk, D, page, device="cpu")
    return cache, torch.zeros((B, 2), dtype=torch.int32), torch.ones(B, dtype=torch.int32), torch.zeros((B, 1, Hk, D), dtype=BF)


def test_refusals_of_append():
    cache, ids, lens, k = setup()
    tab = torch.zeros((8, 16))
    ok = dict(cache=cache, k=k, v=k, page_table=ids, kv_lens=lens)
    with pytest.raises(Error, match="must live on the GPU"):
        C.kv_append(**ok)
    for change, text in [
            (dict(page_table=ids.long()), "page_table"), (dict(page_table=ids[0]), "page_table"), (dict(page_table=ids.repeat(1, 2)[:, ::2]), "page_table"),
            (dict(kv_lens=lens.float()), "kv_lens"), (dict(kv_lens=lens[:1]), "kv_lens"),
            (dict(k=k[0]), "k/v must be"), (dict(v=k[:, :, :1]), "k/v must be"), (dict(k=k.float(), v=k.float()), "BF16 or F16"), (dict(v=k.half()), "BF16 or F16"),
            (dict(k=k[:, :0], v=k[:, :0]), "empty"), (dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), "k/v must be"),
            (dict(k=k[:, 0], v=k[:, 0], cu_seqlens=torch.zeros(2, dtype=torch.int32)), "cu_seqlens"),
            (dict(q=k[:1]), "q must be"), (dict(q=k.half()), "q must be"), (dict(q_norm=tab[0]), "without q"), (dict(q_out=k), "without q"),
            (dict(k_norm=tab[0]), "weight must be"), (dict(k_norm=torch.zeros(64, dtype=torch.float64)), "weights must be"),
            (dict(q=k, k_norm=torch.zeros(64), q_norm=torch.zeros(64, dtype=BF)), "both the same"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
            (dict(cos=tab), "together"), (dict(cos=tab, sin=tab[:4]), "cos/sin"), (dict(cos=tab[:, :4], sin=tab[:, :4]), "rotated"),
            (dict(cos=torch.zeros((8, 40)), sin=torch.zeros((8, 40))), "rotated"), (dict(cos=tab[:0], sin=tab[:0]), "cos/sin"),
            (dict(cos=tab.double(), sin=tab.double()), "tables must be"),
            (dict(q=k, q_out=k.half()), "output"), (dict(q=k, q_out=torch.zeros((2, 1, 2, 128), dtype=BF)[..., ::2]), "rows of an output"),
            (dict(q=k, q_out=k[:, :, :1].expand(2, 1, 2, 64)), "lie apart")]:
        with pytest.raises(Error, match=text):
            C.kv_append(**{**ok, **change})


def test_refusals_of_the_cache_itself():
    cache, ids, lens, k = setup()
    q = torch.zeros((2, 1, 4, 64), dtype=BF)
    parts = dict(k=cache.k, v=cache.v, k_scale=cache.k_scale, v_scale=cache.v_scale)
    for change in (dict(k=cache.k[0]), dict(v=cache.v.transpose(3, 4).contiguous()), dict(k_scale=cache.k_scale[:1]), dict(v_scale=cache.v_scale.double()),
                   dict(k=cache.k.view(torch.uint8)), dict(k=cache.k.transpose(0, 2).contiguous().transpose(0, 2))):
        for call in (lambda c: C.sdpa_paged(q, c, ids, lens, 0.1), lambda c: C.kv_append(c, k, k, ids, lens)):
            with pytest.raises(Error, match="pages"):
                call(C.KvPages(**{**parts, **change}))
    odd = C.KvPages(*(t.repeat(1, 3, *[1] * (t.dim() - 2)) for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)))
    odd.k, odd.v = odd.k.view(cache.k.dtype), odd.v.view(cache.v.dtype)
    with pytest.raises(Error, match="32, 64, 128"):
        C.sdpa_paged(q, odd, ids, lens, 0.1)
    for args in ((0, 1, 64), (1, 0, 64), (1, 1, 96), (1, 1, 64, 48), (1, 1, 64, 16), (1, 1, 64, 131072)):
        with pytest.raises(Error):
            C.KvPages.empty(*args, device="cpu")
    with pytest.raises(Error):
        cache.dense(ids[0], 65)
    k, v = cache.dense(ids[0], 40)
    assert k.shape == v.shape == (40, 2, 64)


def test_dense_looks_at_the_pages_of_its_tokens_only():
    """A table's further entries need be no pages; one that the tokens do need and that is none gives NaN, and no page in its place."""
    cache = C.KvPages.empty(4, 2, 64, 64, device="cpu")
    for t in (cache.k, cache.v):
        t.view(torch.uint8).copy_(torch.arange(t.numel()).remainder(0x77).to(torch.uint8).view(t.shape))
    table = torch.tensor([2, 0, 99, -7, 2 ** 31 - 1], dtype=torch.int32)
    for n in (0, 1, 64, 65, 128):
        k, v = cache.dense(table, n)
        assert k.shape == v.shape == (n, 2, 64)
        for i in (0, n // 2, n - 1)[:n]:
            at = (int(table[i // 64]), i % 64 // 32)
            assert torch.equal(k[i], cache.k[at].float()[:, i % 32]) and torch.equal(v[i], cache.v[at].float()[..., i % 32])
    k, v = cache.dense(table, 300)
    for t in (k, v):
        assert torch.isfinite(t[:128]).all() and torch.isnan(t[128:]).all()


def test_refusals_of_attention():
    cache, ids, lens, _ = setup()
    q = torch.zeros((2, 1, 4, 64), dtype=BF)
    with pytest.raises(Error, match="must live on the GPU"):
        C.sdpa_paged(q, cache, ids, lens, 0.1)
    for bad, text in ((q[:1], "q must be"), (q[0], "q must be"), (q[..., :32], "q must be"), (q[:, :0], "q must be"), (q.float(), "BF16 or F16"), (q[:, :, :3], "share")):
        with pytest.raises(Error, match=text):
            C.sdpa_paged(bad, cache, ids, lens, 0.1)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(Error, match="scale"):
            C.sdpa_paged(q, cache, ids, lens, scale)


def test_sizes_of_the_c_calls():
    """(Sizes and codes only: nothing runs.)"""
    L = _lib.lib()
    size = L.mi355_sage_paged_workspace_bytes
    # two parts of 16 or 32 rows for each of at most 1024 workgroups
    for B, Hq, Hk, N, D, width, page in ((1, 48, 12, 1, 128, 128, 64), (32, 48, 12, 1, 128, 256, 64), (1, 1, 1, 1, 64, 1, 32), (8, 40, 10, 4, 64, 40, 128), (4, 64, 8, 333, 256, 9, 256)):
        got = size(B, Hq, Hk, N, D, width, page)
        assert 0 < got <= 1024 * 2 * 32 * (D + 2) * 4 + 255 and got % 256 == 0
    for bad in ((0, 4, 2, 1, 64, 2, 32), (1, 4, 3, 1, 64, 2, 32), (1, 4, 2, 1, 96, 2, 32), (1, 4, 2, 1, 64, 2, 48), (1, 4, 2, 1, 64, 1 << 25, 32), (1 << 12, 4, 4, 1, 64, 1 << 17, 32)):
        assert size(*bad) == 0
    if torch.cuda.is_available():
        pytest.skip("made-up pointers: runs only where no device can be reached")
    st = (ctypes.c_int64 * 4)(128, 64, 128, 1)
    p = ctypes.c_void_p(4096)
    append = lambda k=p, pages=4, page=32, width=2, B=1, N=1, Hk=2, D=64, type=0, ks=st, q=None, rot=0, gain=None: L.mi355_sage_kv_append(
        k, p, q, None, p, p, p, p, pages, page, p, 2, width, p, None, B, N, 0, Hk, D, type, ks, st, None, None, 0, 0, 0, 0, None, gain, 0, 1e-6, None, None, 0, rot, 8, 8, 0, None)
    assert append(k=None) == append(pages=0) == append(width=0) == append(B=0) == append(N=0) == append(q=p) == append(rot=16) == append(rot=80) == -1
    assert append(D=96) == append(page=48) == append(type=2) == append(width=1 << 25) == append(N=1 << 30) == append(gain=ctypes.c_void_p(4100)) == -2
    assert append(ks=(ctypes.c_int64 * 4)(128, 64, 128, 2)) == append(ks=(ctypes.c_int64 * 4)(128, 60, 128, 1)) == -2
    paged = lambda q=p, Hq=4, N=1, scale=0.1, type=0, page=32, D=64: L.mi355_sage_sdpa_paged(q, p, p, p, p, p, 4, page, p, 2, 2, p, 1, Hq, 2, N, D, type, scale, st, st, 0, 0, None, p, 1 << 20)
    assert paged(q=None) == paged(Hq=3) == paged(N=0) == paged(scale=0.0) == paged(scale=float("inf")) == -1
    assert paged(type=2) == paged(page=33) == paged(D=32) == -2


def test_workspace_of_paged_attention():
    """Two parts of 16 or 32 rows for each of at most 1024 even shares and, up to 2048 row blocks (blocks of 16 or 32 query rows of a sequence and key head), for a share more of each: the
    most that a call takes, and about what it takes."""
    size = _lib.lib().mi355_sage_paged_workspace_bytes
    for B, Hq, Hk, N, D, width, page in ((32, 64, 8, 16, 128, 64, 64), (64, 64, 32, 1, 128, 64, 64), (64, 32, 32, 1, 64, 9, 32), (128, 16, 16, 1, 64, 9, 32), (129, 16, 16, 1, 64, 9, 32),
                                         (16, 32, 8, 127, 64, 3, 64), (16, 32, 8, 128, 64, 3, 64), (16, 32, 8, 129, 64, 3, 64), (1, 1, 1, 1, 256, 1, 32), (2, 64, 64, 1, 256, 100, 32)):
        rows = 16 if N * Hq // Hk <= 16 else 32
        units = B * Hk * -(-N * Hq // Hk // rows)
        shares = min(1024, -(-units * width * (page // 32) // 8)) + (units if units <= 2048 else 0)
        assert size(B, Hq, Hk, N, D, width, page) == -(-shares * 2 * rows * (D + 2) * 4 // 256) * 256
    assert size(16, 32, 8, 128, 64, 300, 64) == 3072 * 2 * 32 * 66 * 4 and size(16, 32, 8, 129, 64, 300, 64) == 1024 * 2 * 32 * 66 * 4


def test_queries_of_an_append_beyond_32_bits_are_refused():
    """2^29 rows of 8 heads are 2^31 groups of two heads, which the kernel numbers in 32 bits; (sizes and codes only: nothing runs)."""
    if torch.cuda.is_available():
        pytest.skip("made-up pointers: runs only where no device can be reached")
    L, p = _lib.lib(), ctypes.c_void_p(4096)
    st = lambda heads: (ctypes.c_int64 * 4)(0, 64, 64 * heads, 1)
    q, out = ctypes.c_void_p(1 << 20), ctypes.c_void_p(1 << 30)
    call = lambda rows, Hq: L.mi355_sage_kv_append(p, p, q, out, p, p, p, p, 4, 32, p, 2, 2, p, p, 1, rows, Hq, 2, 64, 0, st(2), st(2), st(Hq), st(Hq), 0, 0, 0, 0, None, None, 0, 1e-6,
                                                   None, None, 0, 0, 0, 0, 0, None)
    assert call(1 << 29, 8) == call(1 << 29, 7) == call((1 << 28) + 1, 16) == -2
    for rows, Hq in ((1 << 29, 6), (1 << 28, 14), (1000, 64)):
        assert call(rows, Hq) not in (-1, -2)        # (let through: what fails is the launch)


def test_shares_of_long_lists(tmp_path):
    """share_of: every place in one share, ids beyond the last empty, in lists of up to 2^30 places, whose ids times shares pass 32 bits (paged attention: 1024 even shares, up to 3072 ids)."""
    src = tmp_path / "shares.cpp"
    src.write_text('''
#define __host__
#define __device__
#include "%s/sage_grid.h"
#include <cstdio>
using namespace sage;
int main() {
    const int totals[] = {1, 7, 1023, 1024, 5000, 1 << 20, (1 << 30) - 1, 1 << 30};
    for (int total : totals) {
        const int even = (total + 1023) / 1024, pers[] = {even, even + 1, 1 << 20, 1 << 30};
        for (int per : pers) {
            long long at = 0;
            for (int id = 0; id < 3072; id++) {
                const Share s = share_of(id, per, total);
                if (s.begin != at || s.end < s.begin || s.end > total || s.end - s.begin > per) return 1;
                if (s.end < total && s.end - s.begin != per) return 2;
                at = s.end;
            }
            if (at != total) return 3;
        }
    }
    std::puts("ok");
}
''' % CSRC)
    exe = tmp_path / "shares"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-o", str(exe), str(src)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout == "ok\n"
