"""Timed cases of attention over packed sequences, and of a paged cache in 8 bits: appending to it and attending over it.

A case is a dict of plain values:

  op       append          kv_append: new keys and values, normalised and rotated, into a paged cache of e4m3 codes (and the queries rotated beside them)
           paged           sdpa_paged: the last tokens of every sequence against that cache
           packed          sdpa_packed: attention over whole sequences that lie one behind the other
           packed_train    sdpa_packed_train_fwd followed by sdpa_packed_backward: a trainer's step
  B, S     sequences, and the tokens of the longest (append: new tokens; paged: query tokens of each)
  Hq, Hk, D                query heads, key heads, head dim
  dtype    "bf16" or "fp16"
  ragged   sequences of different lengths
  causal   (packed*) a query sees the keys up to itself, else all of its sequence
  cached   (append) tokens that the cache holds already; (paged) tokens of the longest sequence in the cache
  page     tokens to a page
  rot, halfsplit, tables, norm     (append) rotated channels, pairs (i, i + rot/2) instead of (2i, 2i + 1), type of the tables and gains, RMSNorm

A block is 32 tokens of a page.  Its codes of a head share a scale 2^e, the least with which the largest value stays within e4m3's 448 (e at least
-100); while a block fills, its scale only rises, and codes that were there are rounded again to the new one.  Codes: K [pages, blocks of a page, Hk, 32, D],
V [pages, blocks of a page, Hk, D, 32]; scales [pages, blocks of a page, Hk] in fp32.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-6
_BLOCK = 32
_F8 = torch.float8_e4m3fn


def _append(B, S, cached, Hq, Hk, D, dtype, ragged=False, rot=None, halfsplit=True, tables="fp32", norm=True, page=64):
    return {"op": "append", "B": B, "S": S, "cached": cached, "Hq": Hq, "Hk": Hk, "D": D, "dtype": dtype, "ragged": ragged, "rot": D if rot is None else rot,
            "halfsplit": halfsplit, "tables": tables, "norm": norm, "page": page}


def _paged(B, S, cached, Hq, Hk, D, dtype, ragged=False, page=64):
    return {"op": "paged", "B": B, "S": S, "cached": cached, "Hq": Hq, "Hk": Hk, "D": D, "dtype": dtype, "ragged": ragged, "page": page}


def _packed(op, B, S, Hq, Hk, D, dtype, causal=True, ragged=True):
    return {"op": op, "B": B, "S": S, "Hq": Hq, "Hk": Hk, "D": D, "dtype": dtype, "causal": causal, "ragged": ragged}


def listed():
    named = {
        # one new token of 32 served sequences: latency
        "append_token": _append(32, 1, 8191, 48, 12, 128, "bf16"),
        # a batch of new prompts, one behind the other
        "append_prompts": _append(6, 8192, 0, 48, 12, 128, "bf16", ragged=True),
        # a chunk of a few prompts that begins inside a block: head dim 256 of which a quarter is rotated, bf16 tables, no norm
        "append_chunk": _append(3, 1153, 77, 18, 6, 256, "fp16", rot=64, halfsplit=False, tables="bf16", norm=False, page=32),
        # one token of one sequence against its cache: latency
        "paged_token": _paged(1, 1, 8192, 48, 12, 128, "bf16"),
        # a served batch of sequences of different lengths
        "paged_batch": _paged(32, 1, 16384, 48, 12, 128, "bf16", ragged=True),
        # four drafted tokens of eight sequences, odd lengths, narrow heads
        "paged_draft": _paged(8, 4, 4429, 40, 10, 64, "fp16", ragged=True, page=128),
        # a text encoder's batch of captions
        "packed_text": _packed("packed", 16, 333, 12, 12, 64, "fp16"),
        # a batch of long prompts, shared key heads
        "packed_prompts": _packed("packed", 6, 8192, 48, 12, 128, "bf16"),
        # images of different sizes in one batch
        "packed_images": _packed("packed", 4, 4352, 30, 30, 128, "bf16", causal=False),
        # a trainer's step on packed text, shared key heads
        "packed_train_text": _packed("packed_train", 8, 4096, 24, 8, 64, "bf16"),
        # a trainer's step on images of different sizes
        "packed_train_images": _packed("packed_train", 3, 1248, 30, 30, 128, "bf16", causal=False),
    }
    return [dict(c, name=n) for n, c in named.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limit = {}
    for c in listed():
        w = work(c)
        for key in ("bytes", "flops"):
            limit[key] = max(limit.get(key, 0), w[key])
    while True:
        op = rng.choice(["append", "paged", "packed", "packed_train"])
        Hk = rng.choice([1, 2, 3, 4, 6, 8, 10, 12, 18, 30])
        Hq = Hk * rng.choice([1, 1, 2, 3, 4, 5, 8])
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        ragged = rng.random() < 0.6
        page = rng.choice([32, 64, 64, 128, 256])
        if op == "append":
            D = rng.choice([64, 128, 256])
            S = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 8192)])
            case = _append(rng.randint(1, 32), S, rng.choice([0, _log_int(rng, 1, 8192)]), Hq, Hk, D, dtype, ragged, rng.choice([D, D, D // 2, D // 4]),
                           rng.random() < 0.5, rng.choice(["fp32", "fp32", "bf16"]), rng.random() < 0.5, page)
        elif op == "paged":
            case = _paged(rng.randint(1, 32), rng.choice([1, 1, 1, 2, 4, 7]), _log_int(rng, 64, 16384), Hq, Hk, rng.choice([64, 128, 256]), dtype, ragged, page)
        else:
            case = _packed(op, rng.randint(1, 16), _log_int(rng, 17, 8192), Hq, Hk, rng.choice([64, 128, 256] if op == "packed" else [64, 128]), dtype,
                           rng.random() < 0.7, ragged)
        w = work(case)
        if w["bytes"] <= limit["bytes"] and w["flops"] <= limit["flops"] and Hq <= 64:
            return case


def _lens(case, n):
    """Tokens of the sequences: n each, or (ragged) from n down to a bit more than an eighth of it."""
    B = case["B"]
    return [max(1, n - (n * 7 // 8) * b // B) if case["ragged"] else n for b in range(B)]


def _new(case):
    """(append) new tokens of the sequences."""
    return _lens(case, case["S"])


def _cached(case):
    """Tokens in the cache once the call is done (append), or as it begins (paged)."""
    if case["op"] == "append":
        return [n + c if case["cached"] else n for n, c in zip(_new(case), _lens(case, max(case["cached"], 1)))]
    return [max(n, case["S"]) for n in _lens(case, case["cached"])]


def work(case):
    Hq, Hk, D, S = (case[k] for k in ("Hq", "Hk", "D", "S"))
    if case["op"] == "append":
        tokens = sum(_new(case))
        table = min(tokens, max(_cached(case))) * case["rot"] * (4 if case["tables"] == "fp32" else 2)
        return {"bytes": tokens * (4 * Hq * D + 6 * Hk * D) + table, "flops": tokens * ((Hq + Hk) * (4 * D + 3 * case["rot"]) + 4 * Hk * D)}
    if case["op"] == "paged":
        lens = _cached(case)
        blocks = sum(-(-n // _BLOCK) for n in lens)
        return {"bytes": sum(lens) * Hk * 2 * D + 8 * blocks * Hk + 4 * case["B"] * S * Hq * D,
                "flops": 4 * D * Hq * sum(S * (n - S) + S * (S + 1) // 2 for n in lens)}
    lens = _lens(case, S)
    rows, pairs = sum(lens), sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
    q, k = rows * Hq * D * 2, rows * Hk * D * 2
    if case["op"] == "packed_train":             # forward: Q K V in, O and the statistics out; backward: those and dO in, three gradients out
        return {"bytes": 2 * q + 2 * k + 4 * rows * Hq + 4 * q + 4 * k + 4 * rows * Hq, "flops": 14 * pairs * Hq * D}
    return {"bytes": 2 * q + 2 * k, "flops": 4 * pairs * Hq * D}


# ---- inputs ------------------------------------------------------------------------------------------

def _offsets(lens):
    return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def _power(top):
    """The power of two that a block's codes are multiplied by, from its largest value (fp32): the least e with top <= 448 * 2^e, at least -100."""
    m, x = torch.frexp(top)
    return torch.where(top > 0, x - 9 + (m > 0.875), -100).clamp(min=-100)


def _pool(case, g):
    """A page table over a pool with pages to spare, in no order, and a cache full of codes of normal values."""
    B, Hk, D, page = (case[k] for k in ("B", "Hk", "D", "page"))
    width = -(-max(_cached(case)) // page)
    pages, n = B * width + 3, page // _BLOCK
    table = torch.randperm(pages, generator=g, device="cuda")[:B * width].view(B, width).to(torch.int32)
    codes = []
    for _ in range(2):
        x = torch.randn((pages * n * Hk, _BLOCK * D), generator=g, device="cuda")
        e = _power(x.abs().amax(1))
        codes.append((torch.ldexp(x, -e[:, None]).to(_F8).view(pages, n, Hk, _BLOCK * D), torch.ldexp(torch.ones_like(x[:, 0]), e).view(pages, n, Hk)))
    (k, ks), (v, vs) = codes
    return {"table": table, "k_pages": k.view(pages, n, Hk, _BLOCK, D), "v_pages": v.view(pages, n, Hk, D, _BLOCK), "k_scale": ks, "v_scale": vs}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = _TYPES[case["dtype"]]
    B, S, Hq, Hk, D = (case[k] for k in ("B", "S", "Hq", "Hk", "D"))

    def normal(*shape, dtype=t):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    state = {"case": case}
    if case["op"] == "append":
        state |= _pool(case, g)
        state["lens"] = torch.tensor(_cached(case), dtype=torch.int32, device="cuda")
        # the projections of queries, keys and values leave one tensor
        if case["ragged"]:
            state["cu"] = _offsets(_new(case))
            qkv = normal(sum(_new(case)), Hq + 2 * Hk, D)
        else:
            state["cu"] = None
            qkv = normal(B, S, Hq + 2 * Hk, D)
        state["q"], state["k"], state["v"] = qkv[..., :Hq, :], qkv[..., Hq:Hq + Hk, :], qkv[..., Hq + Hk:, :]
        table_type = _TYPES[case["tables"]]
        angle = torch.arange(32768, device="cuda", dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64) * 2 / case["rot"])
        state["cos"], state["sin"] = angle.cos().to(table_type), angle.sin().to(table_type)
        for name in ("q_norm", "k_norm"):
            state[name] = (1 + 0.2 * normal(D, dtype=torch.float32)).to(table_type) if case["norm"] else None
        return state
    if case["op"] == "paged":
        state |= _pool(case, g)
        state["lens"] = torch.tensor(_cached(case), dtype=torch.int32, device="cuda")
        state["q"] = normal(B, S, Hq, D)
        return state
    lens = _lens(case, S)
    # normalised, rotated queries and keys: unit variance, and a direction that the keys share
    state["cu"] = _offsets(lens)
    state["q"], state["k"], state["v"] = normal(sum(lens), Hq, D), normal(sum(lens), Hk, D).add_(0.5 * normal(1, Hk, D)), normal(sum(lens), Hk, D)
    if case["op"] == "packed_train":
        state["d_o"] = normal(sum(lens), Hq, D)
    return state


def run(state):
    case = state["case"]
    return _OWN[case["op"]](state, case) if own else _PLAIN[case["op"]](state, case)


# ---- the framework's calls -----------------------------------------------------------------------

def _own_append(s, c):
    from mojodiffusion_amd import kv_cache as C
    q = C.kv_append(C.KvPages(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]), s["k"], s["v"], s["table"], s["lens"], cu_seqlens=s["cu"],
                    k_norm=s["k_norm"], eps=_EPS, cos=s["cos"], sin=s["sin"], halfsplit=c["halfsplit"], q=s["q"], q_norm=s["q_norm"])
    return q, s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]


def _own_paged(s, c):
    from mojodiffusion_amd import kv_cache as C
    return C.sdpa_paged(s["q"], C.KvPages(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]), s["table"], s["lens"], c["D"] ** -0.5)


def _own_packed(s, c):
    from mojodiffusion_amd import attention_packed as P
    return P.sdpa_packed(s["q"], s["k"], s["v"], s["cu"], c["D"] ** -0.5, causal=c["causal"])


def _own_packed_train(s, c):
    from mojodiffusion_amd import attention_packed as P
    fwd = P.sdpa_packed_train_fwd(s["q"], s["k"], s["v"], s["cu"], c["D"] ** -0.5, causal=c["causal"])
    g = P.sdpa_packed_backward(fwd, s["d_o"])
    return fwd.o, fwd.stats, g.d_q, g.d_k, g.d_v


# ---- the plain forms -------------------------------------------------------------------------------

def _rotate(x, cos, sin, rot, halfsplit):
    if halfsplit:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., rot:]), dim=-1)
    a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    return torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2), x[..., rot:]), dim=-1)


def _norm_rotate(x, gain, cos, sin, c):
    f = x.float()
    if gain is not None:
        f = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + _EPS) * gain.float()
    return _rotate(f, cos, sin, c["rot"], c["halfsplit"])


def _plain_append(s, c):
    B, Hk, D, page = (c[k] for k in ("B", "Hk", "D", "page"))
    lens = s["lens"].long()
    k, v = s["k"].reshape(-1, Hk, D), s["v"].reshape(-1, Hk, D)
    # sequence and position of every token, the block and the row it goes to
    cu = s["cu"].long() if s["cu"] is not None else torch.arange(B + 1, device=k.device) * c["S"]
    token = torch.arange(k.shape[0], device=k.device)
    b = torch.searchsorted(cu, token, right=True) - 1
    start = lens - (cu[1:] - cu[:-1])
    pos = start[b] + token - cu[b]
    cos, sin = s["cos"][pos].float()[:, None], s["sin"][pos].float()[:, None]
    q = _norm_rotate(s["q"].reshape(-1, c["Hq"], D), s["q_norm"], cos, sin, c).to(s["q"].dtype).view(s["q"].shape)
    k, v = _norm_rotate(k, s["k_norm"], cos, sin, c), v.float()
    block = s["table"].long()[b, pos // page] * (page // _BLOCK) + pos % page // _BLOCK
    row = pos % _BLOCK
    used, place = torch.unique(block, return_inverse=True)
    # the row of a block's first new token: earlier ones hold codes
    first = torch.full(used.shape, _BLOCK, device=k.device).scatter_reduce_(0, place, row, "amin")
    kept = torch.arange(_BLOCK, device=k.device) < first[:, None]
    for x, codes, scale, across in ((k, s["k_pages"], s["k_scale"], False), (v, s["v_pages"], s["v_scale"], True)):
        codes, scale = codes.view(torch.uint8).flatten(0, 1), scale.flatten(0, 1)
        top = torch.zeros((used.shape[0], Hk), device=k.device)
        top.scatter_reduce_(0, place[:, None].expand(-1, Hk), x.abs().amax(-1), "amax")
        e, old = _power(top), torch.frexp(scale[used])[1] - 1
        e = torch.where(first[:, None] > 0, torch.maximum(e, old), e)
        rows = codes[used].view(_F8).float()
        rows = rows.transpose(2, 3) if across else rows
        again = torch.ldexp(rows, (old - e)[:, :, None, None]).to(_F8).view(torch.uint8)
        was = codes[used].transpose(2, 3) if across else codes[used]
        again = torch.where(kept[:, None, :, None], again, was)
        again[place, :, row] = torch.ldexp(x, -e[place][:, :, None]).to(_F8).view(torch.uint8)
        codes[used] = again.transpose(2, 3) if across else again
        scale[used] = torch.ldexp(torch.ones_like(top), e)
    return q, s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]


def _softmax(sc):
    """Weights and their log-sum-exp over the last axis."""
    top = sc.amax(-1, keepdim=True)
    e = torch.exp(sc - top)
    total = e.sum(-1, keepdim=True)
    return e / total, torch.log(total) + top


def _plain_paged(s, c):
    q, lens = s["q"], s["lens"].long()
    B, S, Hq, D = q.shape
    Hk, n = c["Hk"], c["page"] // _BLOCK
    o = torch.empty_like(q)
    for b in range(B):
        pages = s["table"][b].long()
        k = (s["k_pages"][pages].float() * s["k_scale"][pages][..., None, None]).permute(2, 0, 1, 3, 4).reshape(Hk, -1, D)
        v = (s["v_pages"][pages].float() * s["v_scale"][pages][..., None, None]).permute(2, 0, 1, 4, 3).reshape(Hk, -1, D)
        j = torch.arange(k.shape[1], device=q.device)
        hidden = j > (lens[b] - S + torch.arange(S, device=q.device))[:, None]
        qb = q[b].float().transpose(0, 1).reshape(Hk, -1, D)                        # the heads that share keys stand together
        p, _ = _softmax((torch.matmul(qb, k.transpose(1, 2).contiguous()) * D ** -0.5).masked_fill_(hidden.repeat(Hq // Hk, 1), float("-inf")))
        o[b] = torch.matmul(p, v).view(Hq, S, D).transpose(0, 1)
    return o


def _plain_packed(s, c, grads=False):
    q, k, v = s["q"], s["k"], s["v"]
    T, Hq, D = q.shape
    Hk, group, scale = c["Hk"], Hq // c["Hk"], D ** -0.5
    o = torch.empty_like(q)
    stats = torch.empty((Hq, T), device=q.device)
    dq, dk, dv = (torch.empty_like(x) if grads else None for x in (q, k, v))
    at = 0
    for n in _lens(c, c["S"]):
        rows = slice(at, at + n)
        at += n
        qb = q[rows].float().transpose(0, 1)
        kb, vb = (x[rows].float().transpose(0, 1).repeat_interleave(group, dim=0) for x in (k, v))
        sc = torch.matmul(qb, kb.transpose(1, 2).contiguous()) * scale
        if c["causal"]:
            j = torch.arange(n, device=q.device)
            sc.masked_fill_(j > j[:, None], float("-inf"))
        p, lse = _softmax(sc)
        ob = torch.matmul(p, vb)
        o[rows], stats[:, rows] = ob.transpose(0, 1), lse[..., 0]
        if grads:
            gb = s["d_o"][rows].float().transpose(0, 1)
            ds = p * (torch.matmul(gb, vb.transpose(1, 2).contiguous()) - (gb * ob).sum(-1, keepdim=True)) * scale
            dq[rows] = torch.matmul(ds, kb).transpose(0, 1)
            dk[rows] = torch.matmul(ds.transpose(1, 2).contiguous(), qb).view(Hk, group, n, D).sum(1).transpose(0, 1)
            dv[rows] = torch.matmul(p.transpose(1, 2).contiguous(), gb).view(Hk, group, n, D).sum(1).transpose(0, 1)
    return (o, stats, dq, dk, dv) if grads else o


_OWN = {"append": _own_append, "paged": _own_paged, "packed": _own_packed, "packed_train": _own_packed_train}
_PLAIN = {"append": _plain_append, "paged": _plain_paged, "packed": _plain_packed, "packed_train": lambda s, c: _plain_packed(s, c, True)}


# ---- from the definitions, in 64 bits ----------------------------------------------------------------

def _e4m3(x):
    """x in 64 bits to the nearest value of e4m3, ties to even: four significant bits, steps of 2^-9 at the least."""
    step = torch.exp2((torch.frexp(x)[1].double() - 4).clamp(min=-9))
    return torch.round(x / step) * step


def _exact_append(s, c):
    """Sequence by sequence, block by block of tokens."""
    Hk, D, rot, n = c["Hk"], c["D"], c["rot"], c["page"] // _BLOCK
    idx = torch.arange(rot // 2, device="cuda")
    ia, ib = (idx, idx + rot // 2) if c["halfsplit"] else (2 * idx, 2 * idx + 1)

    def rows(x, gain, pos):
        x = x.double()
        if gain is not None:
            x = x * gain.double() / (x.square().mean(-1, keepdim=True) + _EPS).sqrt()
        z = x.clone()
        cos, sin = s["cos"][pos].double()[:, None], s["sin"][pos].double()[:, None]
        z[..., ia] = x[..., ia] * cos - x[..., ib] * sin
        z[..., ib] = x[..., ib] * cos + x[..., ia] * sin
        return z

    pages = {"k": s["k_pages"].double(), "v": s["v_pages"].double().transpose(3, 4).contiguous()}
    scales = {"k": s["k_scale"].double(), "v": s["v_scale"].double()}
    q = torch.empty((sum(_new(c)), c["Hq"], D), dtype=torch.float64, device="cuda")
    flat = {x: s[x].reshape(-1, s[x].shape[-2], D) for x in ("q", "k", "v")}
    table, at = s["table"].tolist(), 0
    for b, (new, length) in enumerate(zip(_new(c), _cached(c))):
        pos = torch.arange(length - new, length, device="cuda")
        q[at:at + new] = rows(flat["q"][at:at + new], s["q_norm"], pos)
        fresh = {"k": rows(flat["k"][at:at + new], s["k_norm"], pos), "v": flat["v"][at:at + new].double()}
        at += new
        for block in range((length - new) // _BLOCK, (length - 1) // _BLOCK + 1):
            p0, p1 = max(block * _BLOCK, length - new), min((block + 1) * _BLOCK, length)
            where = (table[b][block // n], block % n)
            for x in ("k", "v"):
                values = fresh[x][p0 - (length - new):p1 - (length - new)].transpose(0, 1)
                top = values.abs().amax((1, 2))
                scale = torch.exp2(torch.ceil(torch.log2(top / 448.0)).clamp(min=-100.0))
                r0 = p0 - block * _BLOCK
                if r0 > 0:
                    old = scales[x][where]
                    scale = torch.maximum(scale, old)
                    pages[x][where][:, :r0] = _e4m3(pages[x][where][:, :r0] * (old / scale)[:, None, None])
                pages[x][where][:, r0:r0 + p1 - p0] = _e4m3(values / scale[:, None, None])
                scales[x][where] = scale
    return q.view(s["q"].shape), pages["k"], pages["v"].transpose(3, 4).contiguous(), scales["k"], scales["v"]


def _exact_attention(q, k, v, seen, scale):
    """One head of one sequence: weights of the visible keys, log-sum-exp, output."""
    sc = torch.where(seen, q @ k.T * scale, -math.inf)
    lse = torch.logsumexp(sc, 1)
    w = torch.exp(sc - lse[:, None])
    return w, lse, w @ v


def _exact_paged(s, c):
    B, S, Hq, D = s["q"].shape
    o = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_cached(c)):
        pages = s["table"][b].long()
        seen = torch.arange(n, device="cuda")[None] <= torch.arange(n - S, n, device="cuda")[:, None]
        for h in range(c["Hk"]):
            k = (s["k_pages"][pages, :, h].double() * s["k_scale"][pages, :, h].double()[..., None, None]).reshape(-1, D)[:n]
            v = (s["v_pages"][pages, :, h].double() * s["v_scale"][pages, :, h].double()[..., None, None]).transpose(2, 3).reshape(-1, D)[:n]
            for hq in range(h * Hq // c["Hk"], (h + 1) * Hq // c["Hk"]):
                o[b, :, hq] = _exact_attention(s["q"][b, :, hq].double(), k, v, seen, 1 / math.sqrt(D))[2]
    return o


def _exact_packed(s, c):
    """Head by head, 2048 queries at a time."""
    q, k, v = s["q"], s["k"], s["v"]
    T, Hq, D = q.shape
    group, train = Hq // c["Hk"], c["op"] == "packed_train"
    o, lse = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros((Hq, T), dtype=torch.float64, device="cuda")
    dq, dk, dv = (torch.zeros(x.shape, dtype=torch.float64, device="cuda") if train else None for x in (q, k, v))
    at = 0
    for n in _lens(c, c["S"]):
        keys = slice(at, at + n)
        for h in range(Hq):
            kh, vh = k[keys, h // group].double(), v[keys, h // group].double()
            for i0 in range(0, n, 2048):
                i1 = min(i0 + 2048, n)
                rows = slice(at + i0, at + i1)
                seen = torch.arange(n, device="cuda")[None] <= (torch.arange(i0, i1, device="cuda")[:, None] if c["causal"] else n)
                qh = q[rows, h].double()
                w, lse[h, rows], o[rows, h] = _exact_attention(qh, kh, vh, seen, 1 / math.sqrt(D))
                if train:
                    gh = s["d_o"][rows, h].double()
                    dw = gh @ vh.T
                    dsc = w * (dw - (w * dw).sum(1, keepdim=True)) / math.sqrt(D)
                    dq[rows, h] = dsc @ kh
                    dk[keys, h // group] += dsc.T @ qh
                    dv[keys, h // group] += w.T @ gh
        at += n
    return (o, lse, dq, dk, dv) if train else o


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s, case)
    if case["op"] == "paged":
        return _exact_paged(s, case)
    # (about 30 operations over every score in 64 bits)
    return _exact_packed(s, case) if case["Hq"] * sum(n * n for n in _lens(case, case["S"])) <= 3e10 else None
