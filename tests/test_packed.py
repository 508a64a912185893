"""Refusals of attention over packed sequences that need no device, its sizes, and how its grid shares slots out."""
import ctypes
import os
import subprocess

import pytest
import torch

from mojodiffusion_amd import _lib
from mojodiffusion_amd import attention_packed as P
from mojodiffusion_amd.attention_sage import Error

BF = torch.bfloat16
CSRC = os.path.join(os.path.dirname(os.path.abspath(_lib.__file__)), "csrc")


def test_refusals():
    q, k = torch.zeros((10, 4, 64), dtype=BF), torch.zeros((10, 2, 64), dtype=BF)
    cu = torch.tensor([0, 4, 10], dtype=torch.int32)
    calls = (P.sdpa_packed, P.sdpa_packed_train_fwd, P.record_sdpa_packed)
    for call in calls:
        with pytest.raises(Error, match="must live on the GPU"):
            call(q, k, k, cu, 0.1)
        for args, text in (((q[None], k, k, cu, 0.1), "rank-3"), ((q, k, k[:, :1], cu, 0.1), "mismatch"), ((q.float(), k, k, cu, 0.1), "BF16 or F16"), ((q, k.half(), k, cu, 0.1), "BF16 or F16"),
                           ((q, k[:9], k[:9], cu, 0.1), "disagree"), ((q, k[..., :32], k[..., :32], cu, 0.1), "disagree"), ((q[:0], k[:0], k[:0], cu, 0.1), "empty"),
                           ((q[:, :3], k, k, cu, 0.1), "share"), ((q[..., :32], k[..., :32], k[..., :32], cu, 0.1), "Dh=32"), ((q, k, k, cu, 0.0), "scale"),
                           ((q, k, k, cu, float("nan")), "scale"), ((q, k, k, cu.float(), 0.1), "cu_seqlens"), ((q, k, k, cu[:1], 0.1), "cu_seqlens"),
                           ((q, k, k, cu[None], 0.1), "cu_seqlens"), ((q, k, k, cu, 0.1, True, cu[:2]), "cu_seqlens")):
            with pytest.raises(Error, match=text):
                call(*args)
    wide = torch.zeros((10, 2, 256), dtype=BF)
    with pytest.raises(Error, match="Dh=256"):
        P.record_sdpa_packed(wide, wide, wide, cu, 0.1)
    f = P.SdpaPackedFwd(q, q, torch.zeros((4, 10)), q, k, k, cu, None, 0.1, True)
    for d, text in ((q.half(), "type"), (q[:, :2], "shape"), (q, "must live on the GPU")):
        with pytest.raises(Error, match=text):
            P.sdpa_packed_backward(f, d)
    for change, text in ((dict(stats=torch.zeros((4, 9))), "stats"), (dict(o_rest=q[:5]), "shape"), (dict(scale=-1.0), "scale")):
        with pytest.raises(Error, match=text):
            P.sdpa_packed_backward(P.SdpaPackedFwd(**{**f.__dict__, **change}), q)


def test_sizes_and_codes_of_the_c_calls():
    """(Sizes and codes only: nothing runs.)"""
    L = _lib.lib()
    size = L.mi355_sage_packed_bwd_workspace_bytes
    for B, Hq, Hk, T, Tk, D in ((1, 4, 2, 100, 100, 64), (8, 24, 8, 16384, 16384, 64), (3, 30, 30, 2341, 2341, 128), (1, 1, 1, 300000, 300000, 128), (100, 8, 1, 5000, 9000, 128), (1, 64, 1, 1 << 20, 1 << 20, 64)):
        got = size(B, Hq, Hk, T, Tk, D)
        stats = 3 * 4 * Hq * (T + 32 * (B + 1))
        # parts: four for each of 256 compute units at the most, and for every sequence a block that may be empty
        assert 0 < got <= stats + 4 * 256 + (1024 + 1024 * (B + 1)) * 2 * 64 * D * 4
    for bad in ((0, 4, 2, 100, 100, 64), (1, 4, 3, 100, 100, 64), (1, 4, 2, 0, 100, 64), (1, 4, 2, 100, 100, 256), (1, 4, 2, 1 << 30, 100, 64), (1 << 21, 4, 2, 100, 100, 64)):
        assert size(*bad) == 0
    if torch.cuda.is_available():
        pytest.skip("made-up pointers: runs only where no device can be reached")
    st, p = (ctypes.c_int64 * 4)(0, 64, 128, 1), ctypes.c_void_p(4096)
    call = lambda q=p, cu=p, B=1, Hq=2, T=10, D=64, type=0, scale=0.1, qs=st, os=st: L.mi355_sage_sdpa_packed(
        q, p, p, p, None, None, cu, p, B, Hq, 2, T, 10, D, type, scale, qs, st, st, os, 0, 0, 0, 0, 0, 1, None)
    assert call(q=None) == call(cu=None) == call(B=0) == call(Hq=3) == call(T=0) == call(scale=0.0) == call(scale=float("inf")) == call(os=(ctypes.c_int64 * 4)(0, 64, 0, 1)) == -1
    assert call(type=2) == call(D=96) == call(T=1 << 30) == call(B=1 << 21) == call(qs=(ctypes.c_int64 * 4)(0, 64, 100, 1)) == call(qs=(ctypes.c_int64 * 4)(0, 64, 128, 2)) == -2
    bwd = lambda d=p, B=1, D=64, dk=st: L.mi355_sage_sdpa_packed_bwd(
        p, p, p, p, None, d, p, p, p, p, p, p, B, 2, 2, 10, 10, D, 0, 0.1, st, st, st, st, st, st, dk, st, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1, None, p, 1 << 30)
    assert bwd(d=None) == bwd(B=0) == bwd(dk=(ctypes.c_int64 * 4)(0, 64, 0, 1)) == -1 and bwd(D=256) == bwd(D=96) == -2


def test_every_slot_of_every_head_is_somebodys(tmp_path):
    """spread_item: a permutation of (head, slot), with ids beyond the last slot for the rest; and of slots of falling size every XCD gets an even share."""
    src = tmp_path / "spread.cpp"
    src.write_text('''
#define __host__
#define __device__
#include "%s/sage_grid.h"
#include <cstdio>
#include <vector>
using namespace sage;
int main() {
    for (int heads = 1; heads <= 40; heads++)
        for (int slots : {1, 2, 3, 7, 8, 9, 31, 64, 100, 257}) {
            const int n = (int)spread_grid(heads, slots);
            std::vector<int> seen(heads * slots);
            double load[8] = {}, all = 0;
            for (int id = 0; id < n; id++) {
                const HeadSlot at = spread_item(id, heads, slots);
                if (at.head < 0 || at.head >= heads || at.slot < 0) return 1;
                if (at.slot >= slots) continue;
                seen[at.head * slots + at.slot]++;
                load[id & 7] += slots - at.slot, all += slots - at.slot;
            }
            for (int s : seen) if (s != 1) return 2;
            if (n > heads * (slots + 7)) return 3;
            if (slots >= 100)
                for (double l : load) if (l > all / 8 * 1.13 + heads) return 4;
        }
    std::puts("ok");
}
''' % CSRC)
    exe = tmp_path / "spread"
    subprocess.run(["g++", "-O1", "-std=c++17", "-o", str(exe), str(src)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout == "ok\n"


def test_two_waves_to_32_rows_in_one_round_only(tmp_path):
    """packed_form_of, full attention of one long sequence at 128 and 256 channels, where such a workgroup fills a compute unit: never with more than 256 of them; with 129 to 256, always.
    And what the other rows of its table say: causal rows and 64 channels up to 272, few rows in workgroups of 32."""
    src = tmp_path / "form.cpp"
    src.write_text('''
#define __host__
#define __device__
#include "%s/sage_grid.h"
#include <cstdio>
using namespace sage;
int main() {
    for (int D = 64; D <= 256; D *= 2)
        for (int heads = 1; heads <= 40; heads++)
            for (int rows = 1024; rows <= 9000; rows += 31) {
                const int wgs = (rows + 127) / 128 * heads;
                const PackedForm full = packed_form_of(D, false, 1, heads, rows, rows), causal = packed_form_of(D, true, 1, heads, rows, rows);
                if (D > 64 && wgs > 256 && full == PackedForm::kPaired) return std::printf("%%d channels, %%d rows, %%d heads: %%d workgroups\\n", D, rows, heads, wgs), 1;
                if (wgs > 128 + heads && wgs <= 256 && full != PackedForm::kPaired) return 2;
                if (wgs > 128 + heads && wgs <= 272 - heads && causal != PackedForm::kPaired) return 3;
                if ((wgs > 272 + heads && (causal != PackedForm::kFull || full != PackedForm::kFull)) || (wgs <= 64 && (causal != PackedForm::kFew || full != PackedForm::kFew))) return 4;
            }
    // two sequences: rows that whole blocks may make, and others, which make a workgroup more for every head
    if (packed_form_of(128, false, 2, 8, 4096, 2048) != PackedForm::kPaired || packed_form_of(128, false, 2, 8, 4090, 2045) != PackedForm::kFull) return 5;
    std::puts("ok");
}
''' % CSRC)
    exe = tmp_path / "form"
    subprocess.run(["g++", "-O1", "-std=c++17", "-o", str(exe), str(src)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True).stdout == "ok\n"
