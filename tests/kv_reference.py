"""The paged cache of e4m3 codes in float64 on the CPU, from its definition."""
import torch

BLOCK = 32
F8 = torch.float8_e4m3fn


def power(top):
    """The least e with top <= 448 * 2^e, at least -100."""
    e = -100
    while top > 448 * 2.0 ** e:
        e += 1
    return e


def encode(x):
    """Codes of float64 values (already divided by their scale) to the nearest, ties to even; what is not finite: NaN."""
    m, e = torch.frexp(x.abs())
    step = torch.exp2((e.double() - 4).clamp(min=-9))
    y = torch.where(torch.isfinite(x), torch.round(x / step) * step, torch.nan)
    return y.float().to(F8)          # (a value of e4m3: no second rounding)


def rows(x, gain, eps, cos, sin, pos, halfsplit):
    """[n, H, D] normalised and rotated, and a bound on what fp32 makes of it.

    Bound: the mean of squares is a sum of D products (relative error D 2^-24), its root, the reciprocal and two products one step each (6 2^-24 with the
    approximate root's), the rotation two products and a sum, against the pair's size."""
    x = x.double()
    D = x.shape[-1]
    err = torch.zeros_like(x)
    if gain is not None:
        x = x * gain.double() / (x.square().mean(-1, keepdim=True) + eps).sqrt()
        err = x.abs() * (D + 6) * 2.0 ** -24
    z = x.clone()
    if cos is not None:
        r = cos.shape[1]
        i = torch.arange(r)
        a, b = (i, i + r) if halfsplit else (2 * i, 2 * i + 1)
        inside = ((pos >= 0) & (pos < cos.shape[0])).view(-1, 1, 1)
        at = pos.clamp(0, cos.shape[0] - 1)
        c, s = cos.double()[at].unsqueeze(1), sin.double()[at].unsqueeze(1)
        z[..., a] = torch.where(inside, x[..., a] * c - x[..., b] * s, torch.nan)
        z[..., b] = torch.where(inside, x[..., b] * c + x[..., a] * s, torch.nan)
        size = err + 3 * 2.0 ** -24 * x.abs()
        err = err.clone()
        err[..., a] = size[..., a] * c.abs() + size[..., b] * s.abs()
        err[..., b] = size[..., b] * c.abs() + size[..., a] * s.abs()
    return z, err


class Cache:
    """What the pages have to hold, block by block; append() states it, check() compares."""

    def __init__(self, cache):
        self.codes = [cache.k.cpu().clone(), cache.v.cpu().transpose(3, 4).contiguous()]       # both [page, block, head, 32, D]
        self.scale = [cache.k_scale.cpu().clone(), cache.v_scale.cpu().clone()]
        self.value = [torch.full(c.shape, torch.nan, dtype=torch.float64) for c in self.codes]  # of new rows: what the code is the rounding of
        self.err = [torch.zeros(c.shape, dtype=torch.float64) for c in self.codes]
        self.fresh = [torch.zeros(c.shape[:4], dtype=torch.bool) for c in self.codes]

    def append(self, k, v, k_err, pages, start):
        """k, v: [n, H, D] float64, the rows to be stored; start: the first one's position."""
        P, per, H = self.codes[0].shape[:3]
        for x, values, err in ((0, k, k_err), (1, v, torch.zeros_like(v))):
            for p0 in range(start // BLOCK * BLOCK, start + k.shape[0], BLOCK):
                lo, hi = max(start, p0, 0), min(start + k.shape[0], p0 + BLOCK, len(pages) * per * BLOCK)
                if hi <= lo:
                    continue
                page, sub = pages[p0 // (per * BLOCK)], p0 // BLOCK % per
                if not 0 <= page < P:
                    continue
                for h in range(H):
                    new, e_new = values[lo - start:hi - start, h], err[lo - start:hi - start, h]
                    finite = torch.where(torch.isfinite(new), new.abs(), 0.0)
                    top = float(finite.max())
                    got_e = power(top)
                    # (within the bound of a border either power is right)
                    slack = float(torch.where(torch.isfinite(new), e_new, 0.0).max())
                    self.both = {got_e, power(top + slack), power(max(top - slack, 0.0))}
                    e = got_e
                    r0 = lo - p0
                    if r0 > 0:
                        old = int(torch.log2(self.scale[x][page, sub, h]))
                        e = max(e, old)
                        was = self.codes[x][page, sub, h, :r0]
                        self.codes[x][page, sub, h, :r0] = encode(was.double() * 2.0 ** (old - e))
                        assert len({max(b, old) for b in self.both}) == 1, "another seed: a value at a border"
                    else:
                        assert len(self.both) == 1, "another seed: a value at a border"
                    self.scale[x][page, sub, h] = 2.0 ** e
                    self.codes[x][page, sub, h, r0:hi - p0] = encode(new * 2.0 ** -e)
                    self.value[x][page, sub, h, r0:hi - p0] = new
                    self.err[x][page, sub, h, r0:hi - p0] = e_new
                    self.fresh[x][page, sub, h, r0:hi - p0] = True

    def check(self, cache):
        """Scales and codes that are no new row's: the same.  New rows: the nearest code of the value, or the nearest of one as far off as fp32 may be: half a step of
        e4m3 (2^-4 of the value, 2^-10 at the least, times the scale) and that error."""
        got = [cache.k.cpu(), cache.v.cpu().transpose(3, 4).contiguous()]
        for x, scale in ((0, cache.k_scale), (1, cache.v_scale)):
            assert torch.equal(scale.cpu(), self.scale[x])
            same = got[x].view(torch.uint8) == self.codes[x].view(torch.uint8)
            nan = torch.isnan(got[x].float())
            same |= nan & torch.isnan(self.codes[x].float()) & self.fresh[x].unsqueeze(-1)
            assert same[~self.fresh[x]].all()
            if x == 1:
                assert same.all()            # (V goes as it is: no error but the rounding's)
            s = scale.cpu().double()[..., None, None]
            value, new = self.value[x], self.fresh[x].unsqueeze(-1) & ~same
            off = (got[x].double() * s - value).abs()
            bound = torch.maximum(value.abs() * 2.0 ** -4, 2.0 ** -10 * s) + 1.1 * self.err[x]
            assert (off <= bound)[new].all()
