"""The policy-network operators from their definitions, in 64 bits on the host, each with a bound on what a correct
float32 computation rounded to the type may be off by.  U = half a step of float32; a type adds its own half step at
the end.  Bounds are to first order, with every rounding counted at its largest."""
import math

import numpy as np
import torch

U = 2.0 ** -24
TINY = 2.0 ** -126               # the smallest normal number


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """What a result near zero may be off by: half a step of the type's denormals."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def wide(t):
    return None if t is None else t.detach().cpu().double()


# ---- group norm -------------------------------------------------------------------------------------------------
def act_and_slope(z, act, slope):
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    a = {"none": 1.0, "relu": 0.0, "leaky_relu": slope}[act]
    return torch.where(z > 0, z, z * a), torch.where(z > 0, 1.0, a).double()


def group_norm_act(x, groups, weight, bias, eps, act, slope, residual, dy=None):
    """{name: (value, bound)} of y and, given dy, of dx, dresidual, dweight, dbias, for x [n, c, *positions]."""
    t, wt = x.dtype, torch.float32 if weight is None else weight.dtype
    x, r, dy = wide(x), wide(residual), wide(dy)
    n, c = x.shape[:2]
    shape = x.shape
    x = x.reshape(n, groups, c // groups, -1)
    w = (torch.ones(c).double() if weight is None else wide(weight)).reshape(1, groups, -1, 1)
    b = (torch.zeros(c).double() if bias is None else wide(bias)).reshape(1, groups, -1, 1)
    m = x.shape[2] * x.shape[3]
    # a sum of m terms: a thread's own terms one after the other (64 at most at these sizes, were 64 threads to share
    # 4,096), then a tree; k roundings at most on the way of any term
    k = 16 + min(m, 64 + m // 64)
    mean = x.mean((2, 3), keepdim=True)
    var = (x - mean).square().mean((2, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    e_mean = k * U * x.abs().mean((2, 3), keepdim=True)
    # sum (x - mean)^2 with a mean that is e_mean off: + m e_mean^2, and the roundings of terms and sum
    e_var = e_mean.square() + (k + 4) * U * var + 2 * U * (mean.abs() + x.abs().amax((2, 3), keepdim=True)) * torch.sqrt(var)
    e_rstd = rstd * (0.5 * e_var / (var + eps) + 4 * U)
    xh = (x - mean) * rstd
    e_xh = rstd * (e_mean + U * (x - mean).abs() + U * (x.abs() + mean.abs())) + (x - mean).abs() * e_rstd + 2 * U * xh.abs()
    z = xh * w + b
    e_z = e_xh * w.abs() + 3 * U * ((xh * w).abs() + b.abs())
    if r is not None:
        r = r.reshape(x.shape)
        z = z + r
        e_z = e_z + 2 * U * (z.abs() + r.abs())
    y, g = act_and_slope(z, act, slope)
    # silu: |y'| <= 1.1, the exponential and the divisions 8 U and |z| U of the sigmoid, which is 0 where it is below 2^-126 (y = z times
    # it); the others: slope at most 1
    e_y = e_z * 1.1 + (8 + z.abs()) * U * y.abs() + TINY * z.abs() if act == "silu" else e_z + 2 * U * y.abs()
    out = dict(y=(y, e_y + half_step(t) * (y.abs() + e_y) + smallest(t)))
    if dy is not None:
        dy = dy.reshape(x.shape)
        dz = dy * g
        if act == "silu":                            # |y''| <= 0.5
            e_g = 0.5 * e_z + (16 + 2 * z.abs()) * U
        else:                                        # a kink: a z within its error of zero may fall on either side
            a = {"none": 1.0, "relu": 0.0, "leaky_relu": slope}[act]
            e_g = torch.where(z.abs() <= e_z, abs(1 - a), 0.0)
        e_dz = dy.abs() * e_g + 2 * U * dz.abs()
        out["dresidual"] = (dz, e_dz + half_step(t) * (dz.abs() + e_dz) + smallest(t))
        total = n * x.shape[3]
        kk = 16 + min(total, 64 + total // 64 + n)
        e_dzx = e_dz * xh.abs() + dz.abs() * e_xh + 2 * U * (dz * xh).abs()
        for name, v, e in (("dbias", dz, e_dz), ("dweight", dz * xh, e_dzx)):
            s, se = v.sum((0, 3)), e.sum((0, 3)) + kk * U * v.abs().sum((0, 3))
            out[name] = (s, se + half_step(wt) * (s.abs() + se) + smallest(wt))
        dg, e_dg = dz * w, e_dz * w.abs() + 2 * U * (dz * w).abs()
        m1, m2 = dg.mean((2, 3), keepdim=True), (dg * xh).mean((2, 3), keepdim=True)
        e_m1 = e_dg.mean((2, 3), keepdim=True) + (k + 4) * U * dg.abs().mean((2, 3), keepdim=True)
        e_m2 = (e_dzx * w.abs()).mean((2, 3), keepdim=True) + (k + 6) * U * (dg * xh).abs().mean((2, 3), keepdim=True)
        inner = dg - m1 - xh * m2
        e_inner = e_dg + e_m1 + e_xh * m2.abs() + xh.abs() * e_m2 + 4 * U * (dg.abs() + m1.abs() + (xh * m2).abs())
        dx, e_dx = inner * rstd, e_inner * rstd + inner.abs() * e_rstd + 2 * U * (inner * rstd).abs()
        out["dx"] = (dx, e_dx + half_step(t) * (dx.abs() + e_dx) + smallest(t))
    flat = {"dbias": (c,), "dweight": (c,)}
    return {name: (v.reshape(flat.get(name, shape)), e.reshape(flat.get(name, shape))) for name, (v, e) in out.items()}


# ---- dropout ----------------------------------------------------------------------------------------------------
def philox(counter, key):
    """Philox4x32-10 of a 4-tuple of uint64 arrays (or numbers) below 2^32 and a pair of numbers."""
    low = np.uint64(0xFFFFFFFF)
    a, b, c, d = (np.asarray(v, dtype=np.uint64) for v in counter)
    k0, k1 = key
    for _ in range(10):
        p, q = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, d = ((q >> np.uint64(32)) ^ b ^ np.uint64(k0), q & low, (p >> np.uint64(32)) ^ d ^ np.uint64(k1), p & low)
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return a, b, c, d


def threshold(p):
    return int(math.floor(p * 65536 + 0.5))


def keep_mask(n, seed, step, site, p, first=0):
    """Of n elements from block `first` on."""
    blk = np.arange(first, first + (n + 7) // 8, dtype=np.uint64)
    words = philox((blk & np.uint64(0xFFFFFFFF), blk >> np.uint64(32), np.full_like(blk, step & 0xFFFFFFFF),
                    np.full_like(blk, site)), (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    bits = [w & np.uint64(0xFFFF) for w in words] + [w >> np.uint64(16) for w in words]
    return torch.from_numpy((np.stack(bits, 1).reshape(-1)[:n] >= threshold(p)))


def dropout(x, p, seed, step, site, residual=None):
    """(value, bound) in memory order: x, residual [n]."""
    t, n = x.dtype, x.numel()
    thr = threshold(p)
    scale = 0.0 if thr == 65536 else 65536 / (65536 - thr)
    kept = torch.where(keep_mask(n, seed, step, site, p), wide(x).reshape(-1) * scale, 0.0)
    y = kept if residual is None else kept + wide(residual).reshape(-1)
    e = 2 * U * kept.abs() + (0 if residual is None else U * y.abs())     # the scale, the product, the sum
    return y, e + half_step(t) * (y.abs() + e) + smallest(t)


# ---- policy logits ----------------------------------------------------------------------------------------------
def policy_logits(logits, legal=None, bias=None, history=None, history_len=None, repetition=1.0, presence=0.0,
                  frequency=0.0, temperature=1.0, out="logits", dtype=None, dy=None):
    """{name: (value, bound)} of y and, given dy, of dlogits and dbias; legal: truth values [rows, cols]."""
    t = dtype or logits.dtype
    lt, bt = logits.dtype, None if bias is None else bias.dtype
    l, bias64, dy = wide(logits), wide(bias), wide(dy)
    rows, cols = l.shape

    def per_row(v):
        return (wide(v) if torch.is_tensor(v) else torch.full((rows,), float(np.float32(v))).double())[:, None]

    rep, pres, freq, temp = (per_row(v) for v in (repetition, presence, frequency, temperature))
    count = torch.zeros(rows, cols).double()
    if history is not None:
        for i in range(rows):
            h = history[i].cpu()
            if history_len is not None:
                h = h[:max(0, min(len(h), int(history_len[i])))]
            h = h[(h >= 0) & (h < cols)]
            count[i] = torch.bincount(h.long(), minlength=cols).double()
    seen = count > 0
    slope = torch.where(seen, torch.where(l > 0, 1 / rep, rep), 1.0)
    # where nothing is added or scaled nothing is rounded (an infinity stays one and has no error)
    size = lambda v: torch.where(torch.isfinite(v), v.abs(), 0.0)                        # noqa: E731
    a = torch.where(seen, l * slope - pres - freq * count, l)
    e = torch.where(seen, 4 * U * (size(l * slope) + pres.abs() + (freq * count).abs()), 0.0)
    if bias64 is not None:
        a = a + bias64
        e = e + U * size(a)
    z = a / temp
    e = e / temp + 2 * U * size(z)
    off = z == -math.inf
    if legal is not None:
        off = off | ~legal.cpu().bool()
    z, e = torch.where(off, -math.inf, z), torch.where(off, 0.0, e)
    k = 24 + min(cols, 64 + cols // 64)              # roundings on the way of a term of a row's sum
    top = z.amax(1, keepdim=True) if cols else torch.zeros(rows, 1).double()
    top = torch.where(top == -math.inf, 0.0, top)
    w = torch.exp(z - top)
    total = w.sum(1, keepdim=True)
    p = torch.where(off, 0.0, w / total)
    e_far = e + e.amax(1, keepdim=True) + U * size(z - top) if cols else e               # of z - top
    # an exponential: its argument's error, and a rounding of the argument times log2 e
    e_p = p * (e_far + (e_far * p).sum(1, keepdim=True) + (k + 12) * U + 2 * U * size(z - top) * 2)
    # the hardware's exponential has no denormals: w < 2^-126 counts as 0, which takes w / total <= w < 2^-126 from its own p, and
    # from the total less than cols * 2^-126 <= 2^-98 of it (the total is at least 1)
    e_p = e_p + TINY + 2.0 ** -98 * p
    if out == "logits":
        y, e_y = z, e
    elif out == "probs":
        y, e_y = p, e_p
    else:
        lse = torch.log(total)
        y = torch.where(off, -math.inf, z - top - lse)
        e_y = torch.where(off, 0.0, e_far + (e_far * p).sum(1, keepdim=True) + (k + 12) * U + 4 * U * (size(z - top) + size(lse)))
    got = dict(y=(y, e_y + half_step(t) * (size(y) + e_y) + smallest(t)))
    if dy is not None:
        dy = torch.where(off, 0.0, dy)
        if out == "logits":
            dz, e_dz = dy, torch.zeros_like(dy)
        elif out == "log_probs":
            s = dy.sum(1, keepdim=True)
            dz = dy - p * s
            e_s = k * U * dy.abs().sum(1, keepdim=True)
            e_dz = e_p * s.abs() + p * e_s + 2 * U * (dy.abs() + (p * s).abs())
        else:
            s = (p * dy).sum(1, keepdim=True)
            e_s = (e_p * dy.abs()).sum(1, keepdim=True) + (k + 2) * U * (p * dy).abs().sum(1, keepdim=True)
            dz = p * (dy - s)
            e_dz = e_p * (dy - s).abs() + p * (e_s + 3 * U * (dy.abs() + s.abs()))
        dz, e_dz = dz / temp, e_dz / temp + 2 * U * (dz / temp).abs()
        dl = dz * torch.where(off, 0.0, slope)
        e_dl = e_dz * slope + 3 * U * dl.abs()
        got["dlogits"] = (dl, e_dl + half_step(lt) * (dl.abs() + e_dl) + smallest(lt))
        if bias is not None:
            if bias.dim() == 1:
                kk = 16 + min(rows, 64 + rows // 64)
                db, e_db = dz.sum(0), e_dz.sum(0) + kk * U * dz.abs().sum(0)
            else:
                db, e_db = dz, e_dz
            got["dbias"] = (db, e_db + half_step(bt) * (db.abs() + e_db) + smallest(bt))
    return got


def assert_within(got, want, what=""):
    """got (a tensor) against (value, bound); infinities and NaN in the same places."""
    value, bound = want
    got = wide(got).reshape(value.shape)
    odd = ~torch.isfinite(value)
    same = torch.where(torch.isnan(value), torch.isnan(got), got == value)
    assert bool(same[odd].all()), "%s: infinities or NaN in other places" % what
    off = torch.where(odd, 0.0, (got - value).abs()) / torch.where(odd | (bound == 0), 1.0, bound)
    off = torch.where(torch.isnan(off), math.inf, off)
    if off.numel():
        worst = int(off.argmax())
        assert float(off.max()) <= 1.0, "%s: %d of %d values out of bounds, worst at %d: %r, not %r +- %r" % (
            what, int((off > 1).sum()), off.numel(), worst, float(got.reshape(-1)[worst]), float(value.reshape(-1)[worst]),
            float(bound.reshape(-1)[worst]))
