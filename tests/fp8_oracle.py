"""The operators of a feed-forward in 8-bit floating point from their formulas, in 64 bits (torch tensors of either device)."""
import math

import torch

BLOCK = 128
F8 = torch.float8_e4m3fn
TINY = 2.0 ** -126


def e4m3(v):
    """nearest e4m3 value, ties to even, of values up to 448 (1 + 1/30): 464 would be the first that has no nearest one"""
    _, e = torch.frexp(v)
    step = ((e.clamp_min(-5) - 4 + 1023).long() << 52).view(torch.float64)          # (2^(e - 4), exactly)
    return torch.round(v / step) * step


def blocks(n):
    return -(-n // BLOCK)


def per_column(scale, cols):
    return scale.double().repeat_interleave(BLOCK, -1)[..., :cols]


def per_value(scale, rows, cols):
    return per_column(scale.repeat_interleave(BLOCK, -2)[..., :rows, :], cols)


def scales(v):
    """a scale for each 128 columns of a row"""
    return torch.stack([(p.abs().amax(-1) / 448).clamp_min(TINY) for p in v.split(BLOCK, -1)], -1)


def between(q, v, err):
    """whether each q (a value in units of its scale) is what e4m3 makes of some number within err of v"""
    return (e4m3(v - err) <= q) & (q <= e4m3(v + err))


def gated(kind, g, u, limit=7.0):
    if kind == 0:
        return g * torch.sigmoid(g) * u
    if kind == 1:
        return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u
    if kind == 2:
        return g.clamp_min(0) * u
    if kind == 3:
        g, u = g.clamp_max(limit), u.clamp(-limit, limit)
        return g * torch.sigmoid(1.702 * g) * (u + 1)
    return g


def matrix(rows, cols, seed, count=None, std=1.0, device="cuda"):
    """e4m3 values over the whole range (NaN left out) and positive block scales"""
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    lead = () if count is None else (count,)
    q = (60.0 * torch.randn(*lead, rows, cols, generator=g, device=device)).clamp(-448, 448).to(F8)
    s = std / 60.0 * (0.5 + torch.rand(*lead, blocks(rows), blocks(cols), generator=g, device=device))
    return q, s


def quantised(rows, cols, seed, std=1.0, device="cuda"):
    """e4m3 rows and positive scales of their blocks"""
    q, _ = matrix(rows, cols, seed, device=device)
    g = torch.Generator(device=device)
    g.manual_seed(seed + 1)
    return q, std / 60.0 * (0.5 + torch.rand(rows, blocks(cols), generator=g, device=device))


def values(q, s):
    return q.double() * per_column(s, q.shape[-1])


def matrix_values(q, s):
    return q.double() * per_value(s, q.shape[-2], q.shape[-1])


def product(a, sa, w, sw, wide):
    """(rows times the transpose, a bound on the error).  wide: the products of two e4m3 are exact in 32 bits; a block's 128 are added in some order, each addition off by at most a unit in the last
    place (2^-23, truncation allowed) of at most the sum of their sizes; then two products with scales, and the blocks' sums and a few partial sums added up (half a unit, 2^-24, each).  Otherwise
    the matrix cores' 8-bit instructions: of eight products, seven lose what lies below 2^-13 of the largest one, so less than 7 / 2^13 of the sum of their sizes."""
    va, vw = values(a, sa), matrix_values(w, sw)
    size = va.abs() @ vw.abs().transpose(-1, -2)
    return va @ vw.transpose(-1, -2), size * ((0 if wide else 7 * 2.0 ** -13) + 128 * 2.0 ** -23 + (3 + blocks(a.shape[-1]) + 32) * 2.0 ** -24)


def route(score_kind, groups, kept, best_of, renorm, eps, scale, logits, corr, top):
    """row by row, as the words say it"""
    rows, n = logits.shape
    each = n // groups
    idx, wgt = torch.full((rows, top), -1, dtype=torch.int32), torch.zeros(rows, top, dtype=torch.float64)
    z = torch.where(torch.isnan(logits), -math.inf, logits.double())
    score = torch.sigmoid(z) if score_kind == 1 else torch.softmax(z, -1)
    choice = score + (corr.double() if corr is not None else 0.0)
    for t in range(rows):
        c = {e: float(choice[t, e]) for e in range(n) if z[t, e] > -math.inf and not math.isnan(choice[t, e])}
        value = []
        for g in range(groups):
            of = sorted((c[e] for e in range(g * each, (g + 1) * each) if e in c), reverse=True)[:best_of]
            value.append((-sum(of) if of else math.inf, g))
        keep = {g for _, g in sorted(value)[:kept]}
        taken = sorted((-c[e], e) for e in c if e // each in keep)[:top]
        w = [float(score[t, e]) for _, e in taken]
        den = sum(w) + eps
        for k, (_, e) in enumerate(taken):
            idx[t, k] = e
            wgt[t, k] = ((w[k] / den if den > 0 else 0.0) if renorm else w[k]) * scale
    return idx, wgt


def experts(kind, a, sa, gu, sgu, down, sdown, idx, wgt, wide, limit=7.0):
    """(y, a bound on the error; wide: of the second product).  The products' bounds as above.  An activation is off by what its gate and up are off times its slopes (|df/dg| <= 1.2 |u| (kind 3: 1.6 |u + 1|),
    |df/du| <= |f(g, 1)| <= |g|) and 32 roundings of its own evaluation; its e4m3 is then one of those between the ends of that range, and the scale between those of the largest value's."""
    rows, top = idx.shape
    width, ff = a.shape[-1], gu.shape[2]
    y = torch.zeros(rows, width, dtype=torch.float64, device=a.device)
    off, size = torch.zeros_like(y), torch.zeros_like(y)
    for e in range(gu.shape[0]):
        t, k = (idx == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        at, st = a.float()[t], sa[t]
        (g, eg), (u, eu) = (product(at, st, gu[e, i], sgu[e, i], False) for i in (0, 1))
        v = gated(kind, g, u, limit)
        slope = 1.6 * (u.abs() + 1) if kind == 3 else 1.2 * u.abs()
        ev = 1.05 * (eg * (slope + eu) + eu * g.abs()) + 32 * 2.0 ** -24 * v.abs()
        s = scales(v)
        es = torch.stack([p.amax(-1) / 448 for p in ev.split(BLOCK, -1)], -1) + 2.0 ** -23 * s
        f, fe = per_column(s, ff), per_column(es, ff)
        x, ex = v / f, ev / f + v.abs() / f * (fe / f) * 1.05 + 2.0 ** -23 * v.abs() / f
        q = e4m3(x)
        eq = torch.maximum(e4m3((x + ex).clamp(-448, 448)) - q, q - e4m3((x - ex).clamp(-448, 448)))
        d = matrix_values(down[e], sdown[e])
        part, psize = (q * f) @ d.t(), (q * f).abs() @ d.abs().t()
        w = wgt[t, k].double()[:, None]
        y.index_add_(0, t, part * w)
        size.index_add_(0, t, psize * w.abs())
        off.index_add_(0, t, ((eq * f + (q.abs() + eq) * fe) @ d.abs().t() + psize * ((0 if wide else 7 * 2.0 ** -13) + 128 * 2.0 ** -23 + (3 + blocks(ff) + 32) * 2.0 ** -24)) * w.abs())
    return y, off + size * (top + 2) * 2.0 ** -24
