"""The paged cache of e4m3 codes: what an append stores, and attention over it, against float64 (kv_reference, window_reference)."""
import threading

import pytest
import torch

from kv_reference import Cache, rows
from mojodiffusion_amd import kv_cache as C
from mojodiffusion_amd import norm_rope as N
from mojodiffusion_amd.attention_sage import Error
from window_reference import check_forward, forward

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
NAN, INF = float("nan"), float("inf")


def pool(pages, Hk, D, page, seed=0):
    """Pages full of other values: random codes, none a NaN, and scales."""
    g = torch.Generator().manual_seed(seed)
    c = C.KvPages.empty(pages, Hk, D, page)
    for t in (c.k, c.v):
        t.view(torch.uint8).copy_(torch.randint(0, 0x7F, t.shape, generator=g, dtype=torch.uint8) | (torch.randint(0, 2, t.shape, generator=g, dtype=torch.uint8) << 7))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.exp2(torch.randint(-9, -4, t.shape, generator=g).float()))
    return c


def tables(rot, n, dtype):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / rot)
    return a.cos().to(dtype), a.sin().to(dtype)


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


APPEND = [
    # new tokens by sequence (packed, or an int: that many each), lengths after it, Hq, Hk, D, type, page, rot, halfsplit, type of tables and gains, norm
    (1, [1, 32, 33, 8192 % 77, 64], 4, 2, 128, BF, 64, 128, True, F32, True),
    (1, [17], 0, 1, 64, FP, 32, 0, True, F32, False),
    (3, [3, 33, 65, 130, 31], 6, 3, 64, BF, 32, 64, False, BF, True),
    (40, [40, 100, 73], 2, 2, 256, FP, 128, 64, False, F32, True),
    (131, [131, 160], 5, 5, 128, FP, 256, 32, True, FP, False),
    ([1, 0, 70, 33, 32, 5], [1, 9, 70, 90, 64, 37], 9, 3, 128, BF, 64, 128, False, F32, True),
    ([0, 0, 31, 1], [0, 5, 33, 32], 3, 1, 256, BF, 32, 256, True, BF, False),
    ([97, 1, 2], [200, 64, 65], 0, 7, 64, FP, 32, 16, True, FP, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("new,lens,Hq,Hk,D,dtype,page,rot,halfsplit,table,norm", APPEND)
def test_append(new, lens, Hq, Hk, D, dtype, page, rot, halfsplit, table, norm):
    g = torch.Generator().manual_seed(len(lens) * 100 + D + page)
    packed, B = isinstance(new, list), len(lens)
    counts = new if packed else [new] * B
    extra = 3 if packed else 0           # rows behind the last sequence
    T = sum(counts) + extra
    size = torch.exp2(torch.randint(-3, 4, (T, 1, 1), generator=g).float())
    qkv = (torch.randn((T, Hq + 2 * Hk, D), generator=g) * size).to(dtype)
    width = -(-max(lens) // page)
    P = B * width + 2
    table_ids = torch.randperm(P, generator=g)[:B * width].view(B, width).to(torch.int32)
    cos, sin = tables(rot, 260, table) if rot else (None, None)
    gq, gk = (((1 + 0.3 * torch.randn(D, generator=g)).to(table) for _ in range(2)) if norm else (None, None))
    cache = pool(P, Hk, D, page)
    want = Cache(cache)
    at, q_want = 0, []
    for b, n in enumerate(counts):
        part = qkv[at:at + n]
        at += n
        pos = lens[b] - n + torch.arange(n)
        q_want.append(rows(part[:, :Hq], gq, 1e-6, cos, sin, pos, halfsplit))
        k, err = rows(part[:, Hq:Hq + Hk], gk, 1e-6, cos, sin, pos, halfsplit)
        if n:
            want.append(k, part[:, Hq + Hk:].double(), err, table_ids[b].tolist(), lens[b] - n)
    x = qkv.cuda() if packed else qkv.view(B, new, Hq + 2 * Hk, D).cuda()
    q, k, v = x[..., :Hq, :], x[..., Hq:Hq + Hk, :], x[..., Hq + Hk:, :]
    cu = torch.tensor([0] + counts).cumsum(0).to(torch.int32).cuda() if packed else None
    call = lambda c, lens_type, **kw: C.kv_append(c, k, v, table_ids.cuda(), torch.tensor(lens, dtype=lens_type).cuda(), cu_seqlens=cu, k_norm=gk.cuda() if norm else None,
                                                  cos=cos.cuda() if rot else None, sin=sin.cuda() if rot else None, halfsplit=halfsplit,
                                                  q=q if Hq else None, q_norm=gq.cuda() if norm and Hq else None, **kw)
    versions = [t._version for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    got = call(cache, torch.int32)
    assert all(t._version > n for t, n in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), versions))
    want.check(cache)
    if Hq:
        z, err = (torch.cat(t) for t in zip(*q_want))
        flat = got.reshape(T, Hq, D).cpu().double()
        assert (flat[sum(counts):] == 0).all()
        # (fp16's least step is 2^-24)
        assert ((flat[:sum(counts)] - z).abs() <= torch.finfo(dtype).eps / 2 * z.abs() + 1.1 * err + (2.0 ** -25 if dtype == FP else 0)).all()
    else:
        assert got is None
    # again: the same cache; and by the Python path, which takes int64 lengths and an output
    before = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)]
    again = call(cache, torch.int64, **({"q_out": torch.empty_like(got)} if Hq else {}))
    for t, u in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale), before):
        assert torch.equal(t, u)
    assert not Hq or torch.equal(again, got)


@pytest.mark.gpu
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, FP), (256, BF)])
def test_a_block_that_fills_token_by_token(D, dtype):
    """Rising and falling sizes: the scale is that of the largest so far, and codes are what one rounding from the row leaves, or a second one where they fell below
    the normal range (Cache.append does as the definition says, token after token)."""
    g = torch.Generator().manual_seed(D)
    cache = pool(3, 2, D, 32, 1)
    want = Cache(cache)
    ids = torch.tensor([[2, 0]], dtype=torch.int32)
    sizes = [0.01, 0.5, 0.001, 3.0, 40.0, 1e-4, 0.0, 500.0] + [1.0] * 25 + [7.0] * 5
    for i, s in enumerate(sizes):
        k, v = ((s * torch.randn((1, 1, 2, D), generator=g)).to(dtype) for _ in range(2))
        want.append(k[0].double(), v[0].double(), torch.zeros(1, 2, D, dtype=torch.float64), ids[0].tolist(), i)
        C.kv_append(cache, k.cuda(), v.cuda(), ids.cuda(), torch.tensor([i + 1], dtype=torch.int32).cuda())
        want.check(cache)
    k, v = cache.dense(ids[0].cuda(), len(sizes))
    assert k.shape == v.shape == (len(sizes), 2, D) and torch.isfinite(k).all()


@pytest.mark.gpu
def test_values_that_are_not_finite_and_the_ends_of_the_range():
    cache = pool(2, 1, 64, 32)
    want = Cache(cache)
    k, v = torch.randn((1, 20, 1, 64)).to(BF), torch.randn((1, 20, 1, 64)).to(BF)
    k[0, 3, 0, 5], k[0, 4, 0, 6], v[0, 5, 0, 7], v[0, 0, 0, :] = INF, NAN, -INF, NAN
    v[0, 1, 0, 0], k[0, 7, 0, 0] = 3.0e38, 448.0
    want.append(k[0].double(), v[0].double(), torch.zeros(20, 1, 64, dtype=torch.float64), [1], 0)
    C.kv_append(cache, k.cuda(), v.cuda(), torch.tensor([[1]], dtype=torch.int32).cuda(), torch.tensor([20]).cuda())
    want.check(cache)
    # all zeros, and values below the least scale's steps
    small = torch.zeros((1, 4, 1, 64), dtype=BF)
    small[0, 1] = 1e-38
    want.append(small[0].double(), small[0].double(), torch.zeros(4, 1, 64, dtype=torch.float64), [0], 0)
    C.kv_append(cache, small.cuda(), small.cuda(), torch.tensor([[0]], dtype=torch.int32).cuda(), torch.tensor([4]).cuda())
    want.check(cache)
    assert float(cache.k_scale[0, 0, 0]) == 2.0 ** -100
    # a position that the tables do not have: NaN in the rotated channels, and nothing of it in the scale
    cos, sin = tables(32, 3, F32)
    k = torch.randn((1, 5, 1, 64)).to(BF)
    z, err = rows(k[0], None, 0.0, cos, sin, torch.arange(5), True)
    want.append(z, k[0].double(), err, [0], 0)
    C.kv_append(cache, k.cuda(), k.cuda(), torch.tensor([[0]], dtype=torch.int32).cuda(), torch.tensor([5]).cuda(), cos=cos.cuda(), sin=sin.cuda(), halfsplit=True)
    want.check(cache)


@pytest.mark.gpu
def test_tokens_that_have_no_place():
    """Before a sequence's first position, beyond the table, on a page that is none: not stored; everything else is."""
    cache = pool(6, 2, 64, 32)
    want = Cache(cache)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn((5, 40, 2, 64), generator=g).to(FP) for _ in range(2))
    ids = torch.tensor([[0, 1], [2, 9], [-1, 3], [4, 5], [-2 ** 31, 2 ** 31 - 1]], dtype=torch.int32)
    lens = torch.tensor([10, 50, 60, 90, 64], dtype=torch.int32)
    zero = torch.zeros(40, 2, 64, dtype=torch.float64)
    for b in range(4):
        start = int(lens[b]) - 40
        skip = max(0, -start)
        want.append(k[b, skip:].double(), v[b, skip:].double(), zero[skip:], ids[b].tolist(), start + skip)
    C.kv_append(cache, k.cuda(), v.cuda(), ids.cuda(), lens.cuda())
    want.check(cache)
    for n in (-5, 0, -2 ** 31):
        C.kv_append(cache, k.cuda(), v.cuda(), ids.cuda(), torch.full((5,), n, dtype=torch.int32).cuda())
        want.check(cache)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 3, 40])
@pytest.mark.parametrize("packed", [False, True])
def test_lengths_at_the_end_of_32_bits(n, packed):
    """Positions beyond every table: nothing is stored, queries find no row of the tables; a sequence beside them is stored as ever."""
    cache = pool(4, 1, 64, 32)
    want = Cache(cache)
    g = torch.Generator().manual_seed(n)
    q, k, v = (torch.randn((4, n, 1, 64), generator=g).to(BF) for _ in range(3))
    ids = torch.tensor([[0, 1], [2, 3], [2, 3], [2, 3]], dtype=torch.int32)
    lens = torch.tensor([n + 5, 2 ** 31 - 1, 2 ** 40, 2 ** 30 + 7])
    cos, sin = tables(64, 64, F32)
    z, err = rows(k[0], None, 0.0, cos, sin, torch.arange(5, 5 + n), True)
    want.append(z, v[0].double(), err, [0, 1], 5)
    shape = lambda t: (t.reshape(4 * n, 1, 64) if packed else t).cuda()
    cu = torch.arange(5).cuda() * n if packed else None
    got = C.kv_append(cache, shape(k), shape(v), ids.cuda(), lens.cuda(), cu_seqlens=cu, cos=cos.cuda(), sin=sin.cuda(), halfsplit=True, q=shape(q))
    want.check(cache)
    got = got.view(4, n, 1, 64)
    assert torch.isfinite(got[0]).all() and torch.isnan(got[1:]).all()


def filled(lens, Hk, D, page, seed, spare=2):
    """A cache of normal values with pages in no order, its page table, and its values [B, longest, Hk, D] (zeros behind the lengths) in float64."""
    g = torch.Generator().manual_seed(seed)
    B, width = len(lens), -(-max(max(lens), 1) // page)
    cache = C.KvPages.empty(B * width + spare, Hk, D, page)
    ids = torch.randperm(B * width + spare, generator=g)[:B * width].view(B, width).to(torch.int32)
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = torch.randn(codes.shape, generator=g)
        e = torch.randint(-9, -6, scale.shape, generator=g).float()
        codes.copy_((x * torch.exp2(-e - 1)[..., None, None]).clamp(-448, 448).to(torch.float8_e4m3fn))      # (beyond 448 torch's cast gives NaN)
        scale.copy_(torch.exp2(e))
    kv = [torch.zeros((B, max(max(lens), 1), Hk, D)) for _ in range(2)]
    for b, n in enumerate(lens):
        for x, y in zip(kv, cache.dense(ids[b].cuda(), max(n, 0))):
            x[b, :max(n, 0)] = y.cpu()
    return cache, ids.cuda(), kv[0].double(), kv[1].double()


def spoil(cache, ids, lens, page):
    """NaN in every code behind the sequences' lengths, and in every page that no sequence has."""
    ids = ids.cpu()
    used = torch.zeros((*cache.k.shape[:2], 32), dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(0, n):
            used[ids[b, j // page], j % page // 32, j % 32] = True
    u = used.cuda()[:, :, None, :, None]
    cache.k.view(torch.uint8).copy_(torch.where(u, cache.k.view(torch.uint8), 0x7F))
    cache.v.view(torch.uint8).copy_(torch.where(u.transpose(3, 4), cache.v.view(torch.uint8), 0xFF))
    none = (~used.any(2)).cuda()
    cache.k_scale[none], cache.v_scale[none] = NAN, INF


PAGED = [
    # lengths, Sq, Hq, Hk, D, type, page
    ([1], 1, 1, 1, 64, BF, 32),
    ([31, 32, 33, 64, 65], 1, 4, 2, 128, BF, 64),
    ([700, 3, 257], 1, 12, 3, 64, FP, 128),
    ([1000], 1, 16, 1, 128, FP, 32),
    ([257, 1, 0, 90], 1, 10, 5, 256, BF, 256),
    ([2, 300, 1, 0], 4, 8, 2, 128, BF, 32),
    ([5, 129], 7, 6, 2, 64, BF, 64),
    ([40, 7, 520], 7, 8, 1, 128, FP, 64),
    ([333, 50], 20, 5, 1, 256, FP, 32),
    ([150, 260], 50, 6, 3, 64, BF, 128),
    ([2500], 2, 48, 12, 128, BF, 64),
    ([3000], 1, 2, 1, 64, BF, 32),
    ([n * 13 % 190 for n in range(70)], 1, 2, 1, 64, FP, 32),
    ([6000], 1, 3, 1, 256, BF, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,Sq,Hq,Hk,D,dtype,page", PAGED)
def test_attention_over_the_cache(lens, Sq, Hq, Hk, D, dtype, page):
    cache, ids, k, v = filled(lens, Hk, D, page, sum(lens) + D)
    spoil(cache, ids, lens, page)
    g = torch.Generator().manual_seed(D + Sq)
    q = torch.randn((len(lens), Sq, Hq, D), generator=g).to(dtype)
    want = forward(q, k, v, D ** -0.5, -1, 0, 0, lens, [n - Sq for n in lens])
    lens_t = torch.tensor(lens, dtype=torch.int32).cuda()
    o = C.sdpa_paged(q.cuda(), cache, ids, lens_t, D ** -0.5)
    check_forward(o, None, want, dtype)
    for b, n in enumerate(lens):
        assert (o[b, :max(0, Sq - n)] == 0).all()
    # the Python path (int64 lengths; rows of a wider tensor) and again: the same bits
    wide = torch.zeros((len(lens), Sq, Hq + 1, D), dtype=dtype).cuda()
    wide[:, :, 1:] = q.cuda()
    assert torch.equal(C.sdpa_paged(wide[:, :, 1:], cache, ids, lens_t.long(), D ** -0.5), o)
    # a longer table, whose further entries are no pages, may deal the blocks otherwise; the values stay within the bounds
    longer = torch.cat((ids, torch.full((len(lens), 40), -7, dtype=torch.int32).cuda()), 1)
    check_forward(C.sdpa_paged(q.cuda(), cache, longer, lens_t, D ** -0.5), None, want, dtype)


DEALT = [
    # larger lists: rows' own shares of 16 blocks; even shares that straddle rows, by blocks and by more rows than are given their own
    ([9000, 33], 1, 30, 30, 64, FP, 128),
    ([20000, 700], 1, 30, 30, 64, BF, 256),
    ([n * 13 % 97 for n in range(520)], 1, 8, 4, 64, BF, 32),
    ([n * 29 % 300 for n in range(90)], 9, 24, 12, 128, FP, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,Sq,Hq,Hk,D,dtype,page", DEALT)
def test_attention_over_larger_lists(lens, Sq, Hq, Hk, D, dtype, page):
    test_attention_over_the_cache(lens, Sq, Hq, Hk, D, dtype, page)


@pytest.mark.gpu
def test_queries_and_keys_that_are_not_finite():
    lens = [90, 33]
    cache, ids, _, _ = filled(lens, 2, 64, 32, 5)
    q = torch.randn((2, 2, 4, 64)).to(BF).cuda()
    lens_t = torch.tensor(lens, dtype=torch.int32).cuda()
    call = lambda q: C.sdpa_paged(q, cache, ids, lens_t, 0.125)
    want = call(q)
    for bad in (NAN, INF, -INF):
        q2 = q.clone()
        q2[1, 0, 3, 0] = bad
        got = call(q2)
        assert torch.isnan(got[1, 0, 3]).all()
        got[1, 0, 3] = want[1, 0, 3]
        assert torch.equal(got, want)
    # a key that is a NaN: its head's rows that see it (the last of the two), and no others
    cache.k.view(torch.uint8)[ids[0, 2], 0, 1, 89 - 64, 3] = 0x7F
    got = call(q)
    assert torch.isnan(got[0, 1, 2:]).all()
    got[0, 1, 2:] = want[0, 1, 2:]
    assert torch.equal(got, want)
    # a page that is none
    ids[1, 1] = 99
    got = call(q)
    assert torch.isnan(got[1, 1]).all() and torch.equal(got[0, 0], want[0, 0])


@pytest.mark.gpu
def test_lengths_beyond_the_table():
    """A length past the pages of its row counts as what they hold."""
    cache, ids, k, v = filled([64, 64], 2, 64, 32, 7)
    q = torch.randn((2, 3, 4, 64), generator=torch.Generator().manual_seed(1)).to(BF)
    want = C.sdpa_paged(q.cuda(), cache, ids, torch.tensor([64, 64]).cuda(), 0.125)
    check_forward(want, None, forward(q, k, v, 0.125, -1, 0, 0, [64, 64], [61, 61]), BF)
    for lens in ([65, 2 ** 31 - 1], [2 ** 40, 2 ** 30]):
        assert torch.equal(C.sdpa_paged(q.cuda(), cache, ids, torch.tensor(lens).cuda(), 0.125), want)


@pytest.mark.gpu
def test_pages_beyond_32_bit_offsets():
    """9 million blocks of 64 channels: codes of K alone are 18 GB."""
    P = 9_000_000
    cache = C.KvPages.empty(P, 1, 64, 32)
    ids = torch.tensor([[P - 1, 7], [P // 2, P - 2]], dtype=torch.int32).cuda()
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn((2, 50, 1, 64), generator=g).to(BF) for _ in range(2))
    lens = torch.tensor([50, 50], dtype=torch.int32).cuda()
    C.kv_append(cache, k.cuda(), v.cuda(), ids, lens)
    dense = [torch.stack(t).cpu() for t in zip(*(cache.dense(ids[b], 50) for b in range(2)))]
    for x, y in zip(dense, (k, v)):
        assert ((x - y.float()).abs() <= y.float().abs() * 2.0 ** -4 + 2.0 ** -16).all()
    q = torch.randn((2, 1, 2, 64), generator=g).to(BF)
    check_forward(C.sdpa_paged(q.cuda(), cache, ids, lens, 0.125), None, forward(q, *dense, 0.125, -1, 0, 0, [50, 50], [49, 49]), BF)


@pytest.mark.gpu
def test_a_served_batch():
    """Prompts of several lengths, then single tokens: norm, rotation, append and attention, in a captured graph that is replayed, against the same
    steps in float64 from what the cache holds, and against the graph's eager form."""
    B, Hq, Hk, D, steps = 3, 6, 2, 128, 5
    g = torch.Generator().manual_seed(11)
    prompts = [37, 64, 5]
    cos, sin = cuda(*tables(D, 128, F32))
    gq, gk = ((1 + 0.2 * torch.randn(D, generator=g)).cuda() for _ in range(2))
    ids = torch.randperm(12, generator=g)[:9].view(3, 3).to(torch.int32).cuda()
    qkv0 = torch.randn((sum(prompts), Hq + 2 * Hk, D), generator=g).to(BF).cuda()
    tokens = torch.randn((steps, B, 1, Hq + 2 * Hk, D), generator=g).to(BF).cuda()
    parts = lambda x: (x[..., :Hq, :], x[..., Hq:Hq + Hk, :], x[..., Hq + Hk:, :])

    def prefill():
        cache = pool(12, Hk, D, 32, 2)
        q, k, v = parts(qkv0)
        C.kv_append(cache, k, v, ids, torch.tensor(prompts).cuda(), cu_seqlens=torch.tensor([0, 37, 101, 106], dtype=torch.int32).cuda(), k_norm=gk, cos=cos, sin=sin, q=q, q_norm=gq)
        return cache, torch.tensor(prompts, dtype=torch.int32).cuda()

    def step(cache, lens, x):
        lens += 1
        q, k, v = parts(x)
        q = C.kv_append(cache, k, v, ids, lens, k_norm=gk, cos=cos, sin=sin, q=q, q_norm=gq)
        return q, C.sdpa_paged(q, cache, ids, lens, D ** -0.5)

    eager_cache, eager_lens = prefill()
    eager = []
    for x in tokens:
        q, o = step(eager_cache, eager_lens, x)
        lens = eager_lens.tolist()
        kv = [torch.zeros((B, max(lens), Hk, D)) for _ in range(2)]
        for b, n in enumerate(lens):
            for y, z in zip(kv, eager_cache.dense(ids[b], n)):
                y[b, :n] = z.cpu()
        check_forward(o, None, forward(q, *kv, D ** -0.5, -1, 0, 0, lens, [n - 1 for n in lens]), BF)
        # the queries: as qk_norm_rope leaves them, to a rounding
        other = N.qk_norm_rope(parts(x)[0], parts(x)[1], gq, gk, 1e-6, cos, sin, positions=(eager_lens - 1).view(B, 1))[0]
        assert ((q.float() - other.float()).abs() <= 2.0 ** -7 * other.float().abs() + 1e-6).all()
        eager.append(o.clone())
    cache, lens = prefill()
    x = tokens[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        C.sdpa_paged(parts(x)[0], cache, ids, lens, D ** -0.5)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, o = step(cache, lens, x)
    cache2, _ = prefill()
    for a, b in ((cache.k, cache2.k), (cache.v, cache2.v)):
        a.view(torch.uint8).copy_(b.view(torch.uint8))
    cache.k_scale.copy_(cache2.k_scale), cache.v_scale.copy_(cache2.v_scale)
    lens.copy_(torch.tensor(prompts))
    for i in range(steps):
        x.copy_(tokens[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, eager[i]), i
        C.sdpa_paged(parts(x)[0], eager_cache, ids, eager_lens, D ** -0.5)


@pytest.mark.gpu
def test_two_threads_on_streams_of_their_own():
    lens = [500, 900]
    cache, ids, _, _ = filled(lens, 2, 128, 64, 9)
    lens_t = torch.tensor(lens, dtype=torch.int32).cuda()
    qs = [torch.randn((2, 1, 8, 128)).to(BF).cuda() for _ in range(2)]
    want = [C.sdpa_paged(q, cache, ids, lens_t, 0.1) for q in qs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                if not torch.equal(C.sdpa_paged(qs[i], cache, ids, lens_t, 0.1), want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


@pytest.mark.gpu
@pytest.mark.parametrize("D,dtype", [(64, FP), (128, BF), (256, BF)])
def test_other_orders_in_memory(D, dtype):
    """Heads first, rows far apart, rows that are not aligned (copied), tables whose rows are parts of wider ones: the bits of dense tensors."""
    g = torch.Generator().manual_seed(D)
    B, S, Hq, Hk = 2, 37, 4, 2
    q, k, v = (torch.randn((B, S, h, D), generator=g).to(dtype).cuda() for h in (Hq, Hk, Hk))
    ids, lens = torch.tensor([[3, 0, 9], [1, 2, 9]], dtype=torch.int32).cuda()[:, :2], torch.tensor([50, 37], dtype=torch.int32).cuda()
    cos, sin = cuda(*tables(32, 64, F32))
    wide = [torch.cat((t, t), 1)[:, 16:] for t in (cos, sin)]
    gain = (1 + 0.1 * torch.randn(D, generator=g)).cuda()

    def step(q, k, v, cos, sin):
        cache = pool(4, Hk, D, 32, 4)
        z = C.kv_append(cache, k, v, ids, lens, k_norm=gain, cos=cos, sin=sin, halfsplit=True, q=q, q_norm=gain)
        return z, cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale, C.sdpa_paged(q[:, -3:], cache, ids, lens, 0.1)

    want = step(q, k, v, cos, sin)
    heads_first = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)

    def apart(t):
        w = torch.full((B, 2 * S, t.shape[2] + 2, 2 * D), NAN, dtype=dtype, device="cuda")
        w[:, 1::2, 1:-1, D:] = t
        return w[:, 1::2, 1:-1, D:]

    def unaligned(t):
        w = torch.zeros(t.numel() + 1, dtype=dtype, device="cuda")[1:].view(t.shape)
        w.copy_(t)
        return w

    for order in (heads_first, apart, unaligned):
        for table in ((cos, sin), wide):
            for x, y in zip(step(order(q), order(k), order(v), *table), want):
                assert torch.equal(x, y)


@pytest.mark.gpu
def test_q_in_place_and_refusals_on_the_device():
    g = torch.Generator().manual_seed(2)
    cache = pool(4, 2, 64, 32)
    ids, lens = torch.tensor([[0, 1]], dtype=torch.int32).cuda(), torch.tensor([40], dtype=torch.int32).cuda()
    q, k, v = (torch.randn((1, 3, h, 64), generator=g).to(BF).cuda() for h in (4, 2, 2))
    cos, sin = cuda(*tables(64, 64, F32))
    want = C.kv_append(cache, k, v, ids, lens, cos=cos, sin=sin, q=q)
    assert C.kv_append(cache, k, v, ids, lens, cos=cos, sin=sin, q=q, q_out=q) is q and torch.equal(q, want)
    for bad in (lambda: C.kv_append(cache, k, v, ids, lens, q=k, q_out=v), lambda: C.kv_append(cache, k, v, ids.cpu(), lens), lambda: C.sdpa_paged(q, cache, ids, lens.cpu(), 0.1),
                lambda: C.kv_append(cache, k, v, ids, lens, cos=cos, sin=sin, q=q, q_out=q.transpose(0, 1)), lambda: C.sdpa_paged(q, cache, ids, lens, float("nan"))):
        with pytest.raises(Error):
            bad()


def codes(g, *shape):
    """Random codes of every size, none a NaN."""
    return torch.randint(0, 0x7F, shape, generator=g, dtype=torch.uint8) | (torch.randint(0, 2, shape, generator=g, dtype=torch.uint8) << 7)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_one_key_gives_its_value(D, dtype):
    """A row that sees one key is that key's value, code times scale, rounded once: at every scale that the type shows anything of."""
    g = torch.Generator().manual_seed(D)
    for e in (-36, -30, -24, -20, -15, -10, -3, 0, 6, 7):
        cache = C.KvPages.empty(2, 2, D, 32)
        for t in (cache.k, cache.v):
            t.view(torch.uint8).copy_(codes(g, *t.shape))
        cache.k_scale.fill_(2.0 ** -9), cache.v_scale.fill_(2.0 ** e)
        q = torch.randn((2, 1, 6, D), generator=g).to(dtype)
        ids = torch.tensor([[1], [0]], dtype=torch.int32).cuda()
        o = C.sdpa_paged(q.cuda(), cache, ids, torch.tensor([1, 1]).cuda(), D ** -0.5)
        for b in range(2):
            want = cache.dense(ids[b], 1)[1][0].to(dtype)
            assert torch.equal(o[b, 0], want.repeat_interleave(3, 0)), e


def fp16_bound(ref, v, scales):
    """The bound of check_forward with what fp16 loses of small weights as the kernel states it: a weight carries its block's scale and has an absolute step of 2^-25 of the largest
    such product of the row, and meets a code of 448 at the most."""
    O, L, W, A, F, E = ref
    n = W.shape[3]
    largest = (W * scales).amax(3).transpose(1, 2).unsqueeze(-1)
    return 2.0 ** -11 * O.abs() + A * (1.01 * 2.0 ** -11 + n * 2.0 ** -24 + 2.1 * E.transpose(1, 2).unsqueeze(-1)) + n * 448 * 2.0 ** -25 * largest + 2.0 ** -25


@pytest.mark.gpu
@pytest.mark.parametrize("big,small", [(12, -9), (9, -22), (-20, -30)])
def test_fp16_queries_over_values_of_very_different_sizes(big, small):
    """Blocks whose values fp16 cannot hold, or only below its normal range, beside others: rows that do not see them, rows that give them no weight, and rows that see nothing else."""
    D, lens, Sq = 64, [70, 150, 40], 3
    g = torch.Generator().manual_seed(big + 40)
    cache, ids, _, _ = filled(lens, 2, D, 32, 4)
    # the last block of the first two sequences (from key 64, from key 128 on), whose keys point away from the queries in the second; all of the third
    exps = torch.full((3, 150), small, dtype=torch.float64)
    exps[0, 64:], exps[1, 128:], exps[2] = big, big, big
    for b, n in enumerate(lens):
        for j in range(-(-n // 32)):
            cache.v_scale[ids[b, j], 0] = 2.0 ** float(exps[b, j * 32])
    q = (torch.randn((3, Sq, 4, D), generator=g).abs() + 0.5).to(FP)
    k8 = cache.k.view(torch.uint8)
    k8[ids[1, 4].long()] |= 0x80         # (negative codes)
    cache.k_scale[ids[1, 4].long()] = 2.0 ** -4
    kv = [torch.zeros((3, 150, 2, D)) for _ in range(2)]
    for b, n in enumerate(lens):
        for x, y in zip(kv, cache.dense(ids[b], n)):
            x[b, :n] = y.cpu()
    lens[0] = 66                          # (queries at 63, 64, 65: the first does not see the last block)
    ref = forward(q, *kv, D ** -0.5, -1, 0, 0, lens, [n - Sq for n in lens])
    scales = torch.exp2(exps)[:, None, None, :]
    o = C.sdpa_paged(q.cuda(), cache, ids, torch.tensor(lens).cuda(), D ** -0.5).cpu().double()
    # (65504: what is beyond it is an infinity, within the bound of it either is right)
    bound = fp16_bound(ref, kv[1], scales)
    sure = ref[0].abs() + bound < 65504
    assert sure[0, 0].all() and sure[1].all() and torch.isfinite(o[sure]).all()
    assert ((o - ref[0]).abs() <= bound)[sure].all()
    assert (o.abs() >= 32768)[ref[0].abs() - bound > 65536].all()


@pytest.mark.gpu
@pytest.mark.parametrize("D,Sq,Hq", [(64, 1, 2), (128, 4, 6), (256, 1, 16)])
def test_fp16_weights_below_the_normal_range(D, Sq, Hq):
    """One key of every block far above the others, and with a value of zero: what comes out is the sum of the others' weights, 2^-25.5 of the largest each.  Such a weight is off by 2^-32 of
    the largest at the most."""
    n = 1501
    g = torch.Generator().manual_seed(D)
    cache, ids, _, _ = filled([n], 2, D, 32, 1)
    k, v = torch.zeros(cache.k.shape), torch.randint(64, 448, cache.v.shape, generator=g).float()
    k[..., 0, 0], v[..., 0] = 176.0, 0.0
    cache.k.copy_(k.to(torch.float8_e4m3fn)), cache.v.copy_(v.to(torch.float8_e4m3fn))
    cache.k_scale.fill_(1.0), cache.v_scale.fill_(4.0)
    q = torch.zeros((1, Sq, Hq, D), dtype=FP)
    q[..., 0] = 25.5 * 0.6931 / 176 / 2.0 ** -6
    kv = [x[None].cpu() for x in cache.dense(ids[0], n)]
    ref = O, L, W, A, F, E = forward(q, *kv, 2.0 ** -6, -1, 0, 0, [n], [n - Sq])
    assert W[..., 1].max() < 2.0 ** -25.2 * W[..., 0].min() and O.min() > 2.0 ** -12
    bound = 2.0 ** -11 * O.abs() + A * (1.01 * 2.0 ** -11 + n * 2.0 ** -24 + 2.1 * E.transpose(1, 2).unsqueeze(-1)) + n * 448 * 2.0 ** -32 * (4 * W).amax(3).transpose(1, 2).unsqueeze(-1) + 2.0 ** -25
    o = C.sdpa_paged(q.cuda(), cache, ids, torch.tensor([n]).cuda(), 2.0 ** -6).cpu().double()
    assert ((o - O).abs() <= bound).all(), float(((o - O).abs() / bound).max())


@pytest.mark.gpu
def test_values_around_the_least_scale():
    """Half of e4m3's least step at the scale 2^-100 is 2^-110: that and less is zero (to the even code), more is the least step; and larger values as the least scale has them."""
    cache = pool(1, 1, 64, 32)
    x = torch.zeros((1, 3, 1, 64), dtype=BF)
    sizes = [2.0 ** -112, 2.0 ** -111, 1.5 * 2.0 ** -111, 2.0 ** -110, (1 + 2.0 ** -7) * 2.0 ** -110, 1.5 * 2.0 ** -110, 2.0 ** -109, 1.5 * 2.0 ** -109, 2.5 * 2.0 ** -109, 2.0 ** -106, 2.0 ** -92]
    x[0, 0, 0, :11], x[0, 2, 0, 11:22] = torch.tensor(sizes).to(BF), -torch.tensor(sizes).to(BF)
    want = Cache(cache)
    want.append(x[0].double(), x[0].double(), torch.zeros(3, 1, 64, dtype=torch.float64), [0], 0)
    ids = torch.tensor([[0]], dtype=torch.int32).cuda()
    C.kv_append(cache, x.cuda(), x.cuda(), ids, torch.tensor([3]).cuda())
    want.check(cache)
    k, v = cache.dense(ids[0], 3)
    step = 2.0 ** -109
    assert float(cache.k_scale[0, 0, 0]) == 2.0 ** -100 and torch.equal(k, v)
    assert k[0, 0, :11].tolist() == [0, 0, 0, 0, step, step, step, 2 * step, 2 * step, 2.0 ** -106, 2.0 ** -92]


CHUNKS = [
    # some hundred query tokens of every sequence (a prompt's chunk over its cache): row blocks by the hundred, and more than are given shares of their own; more queries than keys
    ([700, 333, 90], 333, 12, 3, 128, BF, 64),
    ([1200], 500, 6, 2, 64, FP, 32),
    ([300, 40], 257, 4, 1, 256, BF, 128),
    ([400, 390, 600, 17], 400, 64, 8, 64, BF, 64),
    ([900, 512], 512, 6, 6, 128, FP, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,Sq,Hq,Hk,D,dtype,page", CHUNKS)
def test_attention_of_a_chunk_over_the_cache(lens, Sq, Hq, Hk, D, dtype, page):
    test_attention_over_the_cache(lens, Sq, Hq, Hk, D, dtype, page)
