"""Timed cases of the operators around windowed attention: the norm and rotation of queries and keys, and attention
over a sliding window with a few first tokens that stay visible.

A case is a dict of plain values:

  op       norm_rope       qk_norm_rope: RMSNorm of every query and key head, then the position rotation
           norm_rope_bwd   qk_norm_rope_backward: gradients of the projections and of both gains
           window          sdpa_window: attention over a sliding window
           window_train    sdpa_window_train_fwd followed by sdpa_window_backward: a trainer's step
           window_decode   sdpa_window_decode: the last tokens of every sequence against a cache
  B, S, Skv, Hq, Hk, D     batch, query tokens, key tokens (length of the cache), query heads, key heads, head dim
  dtype    "bf16", "fp16" or "fp32" (fp32: the norm and rotation only)
  rot      rotated channels of a head (norm_rope*), halfsplit: pairs (i, i + rot/2) instead of (2i, 2i + 1)
  tables   type of the cos / sin tables and of the gains; positions: rows of the tables by token, else by order
  left, right, sinks       a query at position p sees the keys j <= p + right with j >= p - left or j < sinks
                           (left or right -1: no bound on that side)
  ragged   sequences of different lengths, the rest of K and V is padding or not yet written
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-6


def _rope(op, B, S, Hq, Hk, D, dtype, rot=None, halfsplit=True, tables="fp32", positions=False):
    return {"op": op, "B": B, "S": S, "Hq": Hq, "Hk": Hk, "D": D, "dtype": dtype, "rot": D if rot is None else rot, "halfsplit": halfsplit,
            "tables": tables, "positions": positions}


def _window(op, B, S, Skv, Hq, Hk, D, dtype, left, right, sinks, ragged=False):
    return {"op": op, "B": B, "S": S, "Skv": Skv, "Hq": Hq, "Hk": Hk, "D": D, "dtype": dtype, "left": left, "right": right, "sinks": sinks,
            "ragged": ragged}


def listed():
    named = {
        # one new token of eight sequences at their own positions, 48 query and 12 key heads: latency
        "rope_token": _rope("norm_rope", 8, 1, 48, 12, 128, "bf16", positions=True),
        # two images of a DiT sampler's step (256 + 4096 tokens), interleaved pairs
        "rope_image": _rope("norm_rope", 2, 4352, 30, 30, 128, "bf16", halfsplit=False),
        # odd length, head dim 256 of which a quarter is rotated, bf16 tables, fp16 activations
        "rope_partial": _rope("norm_rope", 3, 1153, 18, 6, 256, "fp16", rot=64, tables="bf16"),
        # a LoRA trainer's step at 512x512, two images
        "rope_grad_train": _rope("norm_rope_bwd", 2, 1248, 30, 30, 128, "bf16", halfsplit=False),
        # a long sequence with shared key heads, fp32 activations of a trainer that keeps them
        "rope_grad_long": _rope("norm_rope_bwd", 1, 16896, 40, 10, 64, "fp32", positions=True),
        # a text encoder's local layer: a few hundred tokens, both directions
        "window_text": _window("window", 2, 333, 333, 12, 12, 64, "fp16", 128, 128, 0),
        # local attention of an image's rows, head dim 256, odd length
        "window_wide": _window("window", 1, 4429, 4429, 18, 18, 256, "bf16", 511, 511, 77),
        # prefill of a long prompt, shared key heads, the first tokens kept visible
        "window_prefill": _window("window", 1, 16896, 16896, 48, 12, 128, "bf16", 4095, 0, 4),
        # a trainer's step over local windows, two images
        "window_train_image": _window("window_train", 2, 1248, 1248, 30, 30, 128, "bf16", 256, 256, 0),
        # a trainer's step on a padded batch of long sequences, shared key heads, sinks
        "window_train_text": _window("window_train", 2, 8192, 8192, 24, 8, 64, "bf16", 1023, 0, 4, ragged=True),
        # one token of one sequence against its cache: latency
        "decode_token": _window("window_decode", 1, 1, 8192, 48, 12, 128, "bf16", 1023, 0, 4),
        # a served batch of sequences of different lengths, the window most of the cache
        "decode_batch": _window("window_decode", 32, 1, 16384, 48, 12, 128, "bf16", 8191, 0, 4, ragged=True),
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
        op = rng.choice(["norm_rope", "norm_rope_bwd", "window", "window_train", "window_decode"])
        Hk = rng.choice([1, 2, 3, 4, 6, 8, 12, 18, 30, 40])
        Hq = Hk * rng.choice([1, 1, 2, 3, 4, 5, 8])
        if op.startswith("norm_rope"):
            D = rng.choice([64, 128, 256])
            case = _rope(op, rng.randint(1, 8), _log_int(rng, 1, 16896), Hq, Hk, D, rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                         rng.choice([D, D, D // 2, D // 4]), rng.random() < 0.5, rng.choice(["fp32", "fp32", "bf16"]), rng.random() < 0.5)
        elif op == "window_decode":
            Skv = _log_int(rng, 64, 16384)
            case = _window(op, rng.randint(1, 32), rng.choice([1, 1, 1, 2, 4, 7]), Skv, Hq, Hk, rng.choice([64, 128, 256]),
                           rng.choice(["bf16", "bf16", "fp16"]), rng.choice([-1, _log_int(rng, 16, Skv)]), 0, rng.choice([0, 1, 4, 77]),
                           rng.random() < 0.7)
        else:
            S = _log_int(rng, 65, 16896)
            right = rng.choice([0, 0, _log_int(rng, 16, S)])
            case = _window(op, rng.randint(1, 4), S, S, Hq, Hk, rng.choice([64, 128, 256] if op == "window" else [64, 128]),
                           rng.choice(["bf16", "bf16", "fp16"]), _log_int(rng, 16, S), right, rng.choice([0, 1, 4, 77]), rng.random() < 0.3)
        w = work(case)
        if w["bytes"] <= limit["bytes"] and w["flops"] <= limit["flops"] and Hq <= 64:
            return case


def _lens(case):
    """Lengths of the sequences: all of the buffer, or (ragged) from all of it down to a bit more than half."""
    B, n = case["B"], case["Skv"]
    return [max(1, n - (n // 2) * b // B) if case["ragged"] else n for b in range(B)]


def _first_query(case, n):
    """Position of the first query: the decoded tokens are a sequence's last."""
    return n - case["S"] if case["op"] == "window_decode" else 0


def _pairs(case):
    """Visible (query, key) pairs of one head over the batch, and the keys that any query sees."""
    left = case["left"] if case["left"] >= 0 else 1 << 30
    right = case["right"] if case["right"] >= 0 else 1 << 30
    pairs = keys = 0
    for n in _lens(case):
        p0 = _first_query(case, n)
        for p in range(p0, p0 + case["S"]):
            hi = min(p + right, n - 1)
            lo = max(p - left, 0)
            if p >= 0:
                pairs += max(hi + 1 - lo, 0) + min(case["sinks"], lo, max(hi + 1, 0))
        lo = max(p0 - left, 0)
        keys += n - lo + min(case["sinks"], lo)
    return pairs, keys


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    B, S, Hq, Hk, D = (case[k] for k in ("B", "S", "Hq", "Hk", "D"))
    if case["op"].startswith("norm_rope"):
        rows = B * S * (Hq + Hk)
        table = min(S * (B if case["positions"] else 1), 32768) * case["rot"] * (4 if case["tables"] == "fp32" else 2)
        if case["op"] == "norm_rope":
            return {"bytes": 2 * rows * D * size + table, "flops": rows * (4 * D + 3 * case["rot"])}
        return {"bytes": 3 * rows * D * size + table, "flops": rows * (11 * D + 3 * case["rot"])}
    pairs, keys = _pairs(case)
    row_bytes, key_bytes = B * S * Hq * D * size, keys * Hk * D * size
    if case["op"] == "window_train":             # forward: Q K V in, O and the statistics out; backward: those and dO in, three gradients out
        return {"bytes": 2 * row_bytes + 2 * key_bytes + 4 * B * S * Hq + 4 * row_bytes + 4 * key_bytes + 4 * B * S * Hq,
                "flops": 14 * pairs * Hq * D}
    return {"bytes": 2 * row_bytes + 2 * key_bytes, "flops": 4 * pairs * Hq * D}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = _TYPES[case["dtype"]]
    B, S, Hq, Hk, D = (case[k] for k in ("B", "S", "Hq", "Hk", "D"))

    def normal(*shape, dtype=t):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    if case["op"].startswith("norm_rope"):
        # the projections of queries, keys and values leave one tensor of which the norm takes the first two parts
        qkv = normal(B, S, Hq + 2 * Hk, D)
        table_type = _TYPES[case["tables"]]
        rows = 32768 if case["positions"] else S
        angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64) * 2 / case["rot"])
        state = {"case": case, "q": qkv[:, :, :Hq], "k": qkv[:, :, Hq:Hq + Hk],
                 "q_norm": (1 + 0.2 * normal(D, dtype=torch.float32)).to(table_type), "k_norm": (1 + 0.2 * normal(D, dtype=torch.float32)).to(table_type),
                 "cos": angle.cos().to(table_type), "sin": angle.sin().to(table_type), "positions": None}
        if case["positions"]:
            start = torch.randint(0, rows - S + 1, (B, 1), generator=g, device="cuda")
            state["positions"] = (start + torch.arange(S, device="cuda")).to(torch.int32)
        if case["op"] == "norm_rope_bwd":
            state["d_q"], state["d_k"] = normal(B, S, Hq, D), normal(B, S, Hk, D)
        return state
    Skv = case["Skv"]
    # normalised, rotated queries and keys: unit variance, and a direction that the keys share
    shared = 0.5 * normal(B, 1, Hk, D)
    state = {"case": case, "q": normal(B, S, Hq, D), "k": normal(B, Skv, Hk, D).add_(shared), "v": normal(B, Skv, Hk, D), "lens": None}
    if case["ragged"] or case["op"] == "window_decode":
        state["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")
    if case["op"] == "window_train":
        state["d_o"] = normal(B, S, Hq, D)
    return state


def run(state):
    case = state["case"]
    return _OWN[case["op"]](state, case) if own else _PLAIN[case["op"]](state, case)


# ---- the framework's calls -----------------------------------------------------------------------

def _own_norm_rope(s, c):
    from mojodiffusion_amd import norm_rope as N
    return N.qk_norm_rope(s["q"], s["k"], s["q_norm"], s["k_norm"], _EPS, s["cos"], s["sin"], halfsplit=c["halfsplit"], positions=s["positions"])


def _own_norm_rope_bwd(s, c):
    from mojodiffusion_amd import norm_rope as N
    g = N.qk_norm_rope_backward(s["d_q"], s["d_k"], s["q"], s["k"], s["q_norm"], s["k_norm"], _EPS, s["cos"], s["sin"],
                                halfsplit=c["halfsplit"], positions=s["positions"])
    return g.d_q, g.d_k, g.d_q_norm, g.d_k_norm


def _own_window(s, c):
    from mojodiffusion_amd import attention_window as W
    return W.sdpa_window(s["q"], s["k"], s["v"], c["D"] ** -0.5, c["left"], c["right"], c["sinks"], kv_lens=s["lens"])


def _own_window_train(s, c):
    from mojodiffusion_amd import attention_window as W
    fwd = W.sdpa_window_train_fwd(s["q"], s["k"], s["v"], c["D"] ** -0.5, c["left"], c["right"], c["sinks"], kv_lens=s["lens"])
    g = W.sdpa_window_backward(fwd, s["d_o"])
    return fwd.o, fwd.stats, g.d_q, g.d_k, g.d_v


def _own_window_decode(s, c):
    from mojodiffusion_amd import attention_window as W
    return W.sdpa_window_decode(s["q"], s["k"], s["v"], s["lens"], c["D"] ** -0.5, c["left"], c["sinks"])


# ---- the plain forms -------------------------------------------------------------------------------

def _table_rows(s, c):
    """cos and sin of every token, [B or 1, S, 1, rot / 2] in fp32."""
    if s["positions"] is None:
        return s["cos"][:c["S"]].float()[None, :, None], s["sin"][:c["S"]].float()[None, :, None]
    rows = s["positions"].long()
    return s["cos"][rows].float()[:, :, None], s["sin"][rows].float()[:, :, None]


def _rotate(x, cos, sin, rot, halfsplit):
    if halfsplit:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., rot:]), dim=-1)
    a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    return torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2), x[..., rot:]), dim=-1)


def _plain_norm_rope(s, c):
    cos, sin = _table_rows(s, c)
    out = []
    for x, gain in ((s["q"], s["q_norm"]), (s["k"], s["k_norm"])):
        f = x.float()
        y = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + _EPS) * gain.float()
        out.append(_rotate(y, cos, sin, c["rot"], c["halfsplit"]).to(x.dtype))
    return tuple(out)


def _plain_norm_rope_bwd(s, c):
    cos, sin = _table_rows(s, c)
    dx, dgain = [], []
    for d, x, gain in ((s["d_q"], s["q"], s["q_norm"]), (s["d_k"], s["k"], s["k_norm"])):
        f = x.float()
        inv = torch.rsqrt((f * f).mean(-1, keepdim=True) + _EPS)
        unit = f * inv
        dy = _rotate(d.float(), cos, -sin, c["rot"], c["halfsplit"])
        dgain.append((dy * unit).double().sum((0, 1, 2)).float())
        du = dy * gain.float()
        dx.append((inv * (du - unit * (du * unit).mean(-1, keepdim=True))).to(x.dtype))
    return dx[0], dx[1], dgain[0], dgain[1]


def _blocks(case, step):
    """(first query, behind the last, ranges of keys that those queries can see) for runs of `step` queries; positions start at 0."""
    left = case["left"] if case["left"] >= 0 else 1 << 30
    right = case["right"] if case["right"] >= 0 else 1 << 30
    for i0 in range(0, case["S"], step):
        i1 = min(i0 + step, case["S"])
        lo = max(min(i0 - left, case["Skv"]), 0)
        hi = min(i1 + right, case["Skv"])
        first = min(case["sinks"], lo, hi)
        yield i0, i1, first, lo, max(hi, lo)


def _hidden(case, n, rows, cols):
    """True where the query at position rows[i] does not see key cols[j] of a sequence of n keys."""
    r, k = rows[:, None], cols[None, :]
    seen = (k < n) & (k < case["sinks"] if case["left"] >= 0 else k >= 0) | (k < n) & (k >= r - (case["left"] if case["left"] >= 0 else 1 << 30))
    if case["right"] >= 0:
        seen = seen & (k <= r + case["right"])
    return ~seen


def _probabilities(q, k, hidden, scale):
    """Softmax over the visible keys (a row that sees none: zeros) and its log-sum-exp; q [H,n,D], k [H,m,D]."""
    sc = torch.matmul(q, k.transpose(1, 2).contiguous()) * scale
    sc = sc.masked_fill_(hidden, float("-inf"))
    top = sc.amax(-1, keepdim=True)
    e = torch.exp(sc - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total), torch.log(total) + torch.where(total == 0, torch.zeros_like(top), top)


def _heads(x, group):
    """[n, Hk, D] of any type -> fp32 [Hk * group, n, D], every head `group` times."""
    return x.float().transpose(0, 1).repeat_interleave(group, dim=0)


def _plain_window(s, c, grads=False):
    q, k, v = s["q"], s["k"], s["v"]
    B, S, Hq, D = q.shape
    Hk, group, scale = c["Hk"], Hq // c["Hk"], D ** -0.5
    o = torch.empty_like(q)
    stats = torch.empty((B, Hq, S, 1), device=q.device, dtype=torch.float32)
    dq = torch.empty_like(q) if grads else None
    dk, dv = (torch.zeros((B, Hk, c["Skv"], D), device=q.device) if grads else None for _ in range(2))
    step = max(64, min(1024, (1 << 28) // (Hq * min(c["Skv"], (c["left"] if c["left"] >= 0 else c["Skv"]) + max(c["right"], 0) + 1024))))
    for b in range(B):
        n = c["Skv"] if s["lens"] is None else s["lens"][b]
        for i0, i1, first, lo, hi in _blocks(c, step):
            cols = torch.cat((torch.arange(first, device=q.device), torch.arange(lo, hi, device=q.device)))
            hidden = _hidden(c, n, torch.arange(i0, i1, device=q.device), cols)
            qb = q[b, i0:i1].float().transpose(0, 1)
            kb, vb = (_heads(torch.cat((x[b, :first], x[b, lo:hi])), group) for x in (k, v))
            p, lse = _probabilities(qb, kb, hidden, scale)
            ob = torch.matmul(p, vb)
            o[b, i0:i1] = ob.transpose(0, 1)
            stats[b, :, i0:i1] = lse
            if grads:
                gb = s["d_o"][b, i0:i1].float().transpose(0, 1)
                dp = torch.matmul(gb, vb.transpose(1, 2).contiguous())
                ds = p * (dp - (gb * ob).sum(-1, keepdim=True)) * scale
                dq[b, i0:i1] = torch.matmul(ds, kb).transpose(0, 1)
                for total, left_side, right_side in ((dk, ds, qb), (dv, p, gb)):
                    part = torch.matmul(left_side.transpose(1, 2).contiguous(), right_side).view(Hk, group, -1, D).sum(1)
                    total[b, :, :first] += part[:, :first]
                    total[b, :, lo:hi] += part[:, first:]
    if not grads:
        return o
    return o, stats, dq, dk.transpose(1, 2).to(q.dtype), dv.transpose(1, 2).to(q.dtype)


def _plain_window_decode(s, c):
    q, k, v, lens = s["q"], s["k"], s["v"], s["lens"]
    B, S, Hq, D = q.shape
    o = torch.empty_like(q)
    cols = torch.arange(c["Skv"], device=q.device)
    for b in range(B):
        rows = lens[b] - S + torch.arange(S, device=q.device)
        hidden = _hidden(c, lens[b], rows, cols)
        qb = q[b].float().transpose(0, 1).reshape(c["Hk"], -1, D)                  # the heads that share keys stand together
        p, _ = _probabilities(qb, k[b].float().transpose(0, 1), hidden.repeat(Hq // c["Hk"], 1), D ** -0.5)
        o[b] = torch.matmul(p, v[b].float().transpose(0, 1).contiguous()).view(Hq, S, D).transpose(0, 1)
    return o


_OWN = {"norm_rope": _own_norm_rope, "norm_rope_bwd": _own_norm_rope_bwd, "window": _own_window, "window_train": _own_window_train,
        "window_decode": _own_window_decode}
_PLAIN = {"norm_rope": _plain_norm_rope, "norm_rope_bwd": _plain_norm_rope_bwd, "window": _plain_window,
          "window_train": lambda s, c: _plain_window(s, c, True), "window_decode": _plain_window_decode}


# ---- from the definitions, in 64 bits ----------------------------------------------------------------

def _exact_rows(x, gain, d, cos, sin, case):
    """One of Q and K, a row at a time as a matrix times a vector: y = x g / sqrt(mean x^2 + eps), z = R y with the rotation
    R = cos on the diagonal and -sin / sin at the pairs; gradients by the chain rule of the quotient."""
    x, gain = x.double(), gain.double()
    D, rot = case["D"], case["rot"]
    idx = torch.arange(rot // 2, device=x.device)
    a, b = (idx, idx + rot // 2) if case["halfsplit"] else (2 * idx, 2 * idx + 1)
    power = x.square().sum(-1, keepdim=True) / D + _EPS
    if d is None:
        z = x * gain / power.sqrt()
        ya, yb = z[..., a], z[..., b]
        z[..., a], z[..., b] = ya * cos - yb * sin, yb * cos + ya * sin
        return z
    dy = d.double().clone()
    za, zb = dy[..., a], dy[..., b]
    dy[..., a], dy[..., b] = za * cos + zb * sin, zb * cos - za * sin
    d_gain = (dy * x / power.sqrt()).sum((0, 1, 2))
    inner = (dy * gain * x).sum(-1, keepdim=True)
    return dy * gain / power.sqrt() - x * inner / (D * power * power.sqrt()), d_gain


def _exact_norm_rope(s, c):
    rows = s["positions"].long() if c["positions"] else torch.arange(c["S"], device="cuda").expand(c["B"], c["S"])
    cos, sin = s["cos"].double()[rows].unsqueeze(2), s["sin"].double()[rows].unsqueeze(2)
    if c["op"] == "norm_rope":
        return tuple(_exact_rows(s[n], s[n + "_norm"], None, cos, sin, c) for n in ("q", "k"))
    dq, gq = _exact_rows(s["q"], s["q_norm"], s["d_q"], cos, sin, c)
    dk, gk = _exact_rows(s["k"], s["k_norm"], s["d_k"], cos, sin, c)
    return dq, dk, gq, gk


def _exact_window(s, c):
    """Head by head and query block by query block against all keys of the sequence, hidden ones left out of the sums."""
    q, k, v = s["q"], s["k"], s["v"]
    B, S, Hq, D = q.shape
    group, train = Hq // c["Hk"], c["op"] == "window_train"
    o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros((B, Hq, S, 1), dtype=torch.float64, device="cuda")
    dq = torch.zeros_like(o) if train else None
    dk, dv = (torch.zeros(k.shape, dtype=torch.float64, device="cuda") if train else None for _ in range(2))
    lens = _lens(c)
    for b in range(B):
        n, p0 = lens[b], _first_query(c, lens[b])
        for h in range(Hq):
            kh, vh = k[b, :n, h // group].double(), v[b, :n, h // group].double()
            for i0 in range(0, S, 2048):
                i1 = min(i0 + 2048, S)
                pos = torch.arange(p0 + i0, p0 + i1, device="cuda").view(-1, 1)
                j = torch.arange(n, device="cuda").view(1, -1)
                seen = torch.ones((i1 - i0, n), dtype=torch.bool, device="cuda")
                if c["left"] >= 0:
                    seen &= (pos - j <= c["left"]) | (j < c["sinks"])
                if c["right"] >= 0:
                    seen &= j - pos <= c["right"]
                qh = q[b, i0:i1, h].double()
                sc = qh @ kh.T / math.sqrt(D)
                sc[~seen] = -math.inf
                lse[b, h, i0:i1, 0] = torch.logsumexp(sc, 1)
                empty = ~seen.any(1, keepdim=True)
                w = torch.where(empty, 0.0, torch.exp(sc - lse[b, h, i0:i1]))
                o[b, i0:i1, h] = w @ vh
                if train:
                    gh = s["d_o"][b, i0:i1, h].double()
                    dw = gh @ vh.T
                    dsc = w * (dw - (w * dw).sum(1, keepdim=True)) / math.sqrt(D)
                    dq[b, i0:i1, h] = dsc @ kh
                    dk[b, :n, h // group] += dsc.T @ qh
                    dv[b, :n, h // group] += w.T @ gh
    return (o, lse, dq, dk, dv) if train else o


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("norm_rope"):
        return _exact_norm_rope(s, case)
    # (about 30 operations over every score in 64 bits)
    if case["B"] * case["Hq"] * case["S"] * case["Skv"] > 4e10:
        return None
    return _exact_window(s, case)
