"""Plain evaluations in 64 bits of the attention operators, with first-order bounds of what 32-bit arithmetic may lose."""
import math

import torch

HALF_STEP = {torch.float64: 0.0, torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# below the smallest normal number (half: 2^-14) a type's numbers are a fixed step apart (half: 2^-14 eps = 2^-24), so a
# rounding is off by up to half of that whatever the value
HALF_SUBNORMAL = {torch.float64: 0.0, torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
E32 = 2.0 ** -24
# For 16-bit types the weights enter the second product as the sum of two numbers of the type: the first is off by up to half
# a step, the second holds what is missing up to half a step of that.  The matrix units' sums may drop digits, so that each
# addition is off by a whole step and not by half of one.
SPLIT = {torch.float64: 0.0, torch.float32: 0.0, torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -22}


def random_pattern(gen, m, n, mean, ptr=torch.int64, idx=torch.int32, hub=0, empty=0.2):
    """Degrees around ``mean``, a share of empty rows, row 1 with ``hub`` edges; ids repeat and are in no order."""
    deg = torch.randint(0, 2 * mean + 1, (m,), generator=gen)
    deg[torch.rand(m, generator=gen) < empty] = 0
    if hub and m > 1:
        deg[1] = hub
    rowptr = torch.zeros(m + 1, dtype=ptr)
    rowptr[1:] = torch.cumsum(deg, 0)
    col = torch.randint(0, max(n, 1), (int(deg.sum()),), generator=gen)
    return rowptr, col.to(idx)


def attention_reference(rowptr, colidx, bias, q, k, v, lam, scale, dout=None):
    """Differential attention from its definition, in 64 bits on the CPU.  -> dict name -> (value, bound of the 32-bit error)."""
    c = lambda t: None if t is None else t.detach().cpu().double()
    rowptr, colidx = rowptr.cpu().long(), colidx.cpu().long()
    half, tiny = HALF_STEP[q.dtype], HALF_SUBNORMAL[q.dtype] + 1e-30
    split, E32 = SPLIT[q.dtype], 2.0 ** -24 if q.dtype == torch.float32 else 2.0 ** -23
    q, k, v, lam, bias, dout = c(q), c(k), c(v), c(lam), c(bias), c(dout)
    m, heads, _, d = q.shape
    n, kvh, dv = v.shape
    row = torch.repeat_interleave(torch.arange(m), rowptr[1:] - rowptr[:-1])
    e = torch.arange(int(rowptr[0]), int(rowptr[-1]))
    col = colidx[e]
    keep = (col >= 0) & (col < n)
    if bias is not None:
        keep &= bias[e] > -math.inf
    row, col, e = row[keep], col[keep], e[keep]
    b = torch.zeros(len(e), dtype=torch.float64) if bias is None else bias[e]
    kv = torch.arange(heads) // (heads // kvh)
    lam_rows = lam.expand(m, heads) if lam.dim() == 1 else lam
    qe, ke, ve = q[row], k[col][:, kv], v[col][:, kv]
    zeros = lambda *s: torch.zeros(s, dtype=torch.float64)
    dot = (qe * ke).sum(-1)
    s = scale * dot + b[:, None, None]
    top = torch.full((m, heads, 2), -math.inf, dtype=torch.float64)
    top.scatter_reduce_(0, row[:, None, None].expand_as(s), s, "amax")
    ref = torch.where(top.isinf(), torch.zeros_like(top), top)
    ex = torch.exp(s - ref[row])
    total = zeros(m, heads, 2).index_add(0, row, ex)
    pr = ex / total[row]
    lse = ref + torch.log(total)
    deg = torch.bincount(row, minlength=m).double()
    # a score is a sum of d products, then a product and a sum: each step rounds
    serr = E32 * ((d + 2) * abs(scale) * (qe.abs() * ke.abs()).sum(-1) + 2 * s.abs())
    smax = zeros(m, heads, 2).scatter_reduce(0, row[:, None, None].expand_as(s), serr, "amax")
    # relative error of p: the score's and the sum's (which holds the scores' again), the exponentials' (2 units), the sums'
    perr = 2 * smax + E32 * (16 + deg)[:, None, None]
    perr = perr.amax(-1) + split
    w = pr[..., 0] - lam_rows[row] * pr[..., 1]
    wabs = pr[..., 0] + lam_rows[row].abs() * pr[..., 1]
    out = zeros(m, heads, dv).index_add(0, row, w[..., None] * ve)
    mag = zeros(m, heads, dv).index_add(0, row, wabs[..., None] * ve.abs())
    bound = lambda value, b32, h, low=tiny: h * value.abs() + b32 * (1 + h) + low
    res = {"out": (out, bound(out, perr[..., None] * mag, half)),
           "lse": (lse, 2 * smax + E32 * (16 + deg)[:, None, None] + 2 * E32 * torch.where(lse.isinf(), torch.zeros_like(lse), lse).abs())}
    if dout is None:
        return res
    de = dout[row]
    dp, dpabs = (de * ve).sum(-1), (de.abs() * ve.abs()).sum(-1)
    delta = zeros(m, heads, 2).index_add(0, row, pr * dp[..., None])
    dabs = zeros(m, heads, 2).index_add(0, row, pr * dpabs[..., None])
    sign = torch.stack((torch.ones_like(lam_rows), -lam_rows), -1)[row]
    ds = sign * pr * (dp[..., None] - delta[row])
    dsabs = sign.abs() * pr * (dpabs[..., None] + dabs[row])
    # what a ds loses against its parts' sizes: p, the dot of dv products, the sum over the row
    rel = (2 * perr + split + E32 * (dv + deg + 16)[:, None])[row]
    dq = zeros(m, heads, 2, d).index_add(0, row, scale * ds[..., None] * ke)
    dqb = zeros(m, heads, 2, d).index_add(0, row, abs(scale) * (rel[..., None] * dsabs)[..., None] * ke.abs())
    group = heads // kvh
    fold = lambda t: t.reshape(t.shape[0], kvh, group, *t.shape[2:]).sum(2)
    indeg = torch.bincount(col, minlength=n).double() * group
    crel = rel[..., None] + E32 * (indeg[col] + 2)[:, None, None]
    dk = zeros(n, kvh, 2, d).index_add(0, col, fold(scale * ds[..., None] * qe))
    dkb = zeros(n, kvh, 2, d).index_add(0, col, fold(abs(scale) * (crel * dsabs)[..., None] * qe.abs()))
    dvv = zeros(n, kvh, dv).index_add(0, col, fold(w[..., None] * de))
    dvb = zeros(n, kvh, dv).index_add(0, col, fold((crel[..., 0] * wabs)[..., None] * de.abs()))
    dlam, dlamb = -delta[..., 1], dabs[..., 1] * (perr + E32 * (dv + deg + 16)[:, None])
    if lam.dim() == 1:
        dlamb = (dlamb + E32 * (m / 2048 + 32) * dabs[..., 1]).sum(0)  # rows summed in runs of m/2048, 8 and 256 of them
        dlam = dlam.sum(0)
    res.update(dq=(dq, bound(dq, dqb, half)), dk=(dk, bound(dk, dkb, half)), dv=(dvv, bound(dvv, dvb, half)),
               dlam=(dlam, bound(dlam, dlamb, E32, 1e-30)))
    return res


def rotary_reference(x, w, pos, freq, eps, interleaved, dy=None):
    """Norm and rotation of one tensor [rows, heads, d] in 64 bits on the CPU.  -> dict as above."""
    half, tiny = HALF_STEP[x.dtype], HALF_SUBNORMAL[x.dtype] + 1e-30
    c = lambda t: None if t is None else t.detach().cpu().double()
    x, w, pos, freq, dy = c(x), c(w), c(pos), c(freq), c(dy)
    rows, heads, d = x.shape
    w = torch.ones(d, dtype=torch.float64) if w is None else w
    if eps is not None:
        r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        y = x * r * w
    else:
        r, y = torch.ones(rows, heads, 1, dtype=torch.float64), x
    pairs = 0 if freq is None else freq.shape[-1]
    mat = torch.eye(d, dtype=torch.float64).repeat(rows, 1, 1)  # the turn as a matrix
    if pairs:
        ang = (pos.reshape(rows, -1) @ freq.reshape(-1, pairs)).reshape(rows, pairs)
        i = torch.arange(pairs)
        lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
        mat[:, lo, lo] = torch.cos(ang)
        mat[:, lo, hi] = -torch.sin(ang)
        mat[:, hi, lo] = torch.sin(ang)
        mat[:, hi, hi] = torch.cos(ang)
    # norm: d squares summed, root, two products; a sine off by 4 units of its largest value; two products and a sum
    rel = E32 * (d / 2 + 16)
    out = torch.einsum("rij,rhj->rhi", mat, y)
    mag = torch.einsum("rij,rhj->rhi", (mat != 0).double(), y.abs())
    res = {"y": (out, half * out.abs() + (1 + half) * rel * mag + tiny)}
    if dy is not None:
        g = torch.einsum("rji,rhj->rhi", mat, dy)
        gabs = torch.einsum("rji,rhj->rhi", (mat != 0).double(), dy.abs())
        if eps is None:
            res["dx"] = (g, half * g.abs() + (1 + half) * rel * gabs + tiny)
        else:
            xn = x * r
            dw = (g * xn).sum((0, 1))
            dx = r * (w * g - xn * (w * g * xn).mean(-1, keepdim=True))
            mag = r * ((w * gabs).abs() + xn.abs() * (w.abs() * gabs * xn.abs()).mean(-1, keepdim=True))
            res["dx"] = (dx, half * dx.abs() + (1 + half) * 4 * rel * mag + tiny)
            # weights: every thread adds its rows, then slots, then blocks: no chain is longer than the count of terms
            res["dw"] = (dw, E32 * dw.abs() + (2 * rel + E32 * (rows * heads / 64 + 64)) * (gabs * xn.abs()).sum((0, 1)) + 1e-30)
    return res


def check(got, wanted, name=""):
    value, bound = wanted
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    same = got == value  # equal infinities
    off = torch.where(same, torch.zeros_like(got), (got - value).abs())
    assert bool((off <= bound).all()), f"{name}: off by up to {float((off / bound).max()):.3g} of the bound, {int((off > bound).sum())} values"
