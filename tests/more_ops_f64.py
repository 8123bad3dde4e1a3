"""64-bit statements of the selective scan, the block-scaled fp8 product and sampling, with bounds on what the
library's arithmetic may differ by."""
import math

import numpy as np
import torch

U = 2.0 ** -24                      # half a step of f32, relative
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}
SLACK = 1.01                        # products of two errors, which the bounds leave out


class V:
    """A value in 64 bits and how far one computed in f32 may be off: each operation carries its operands' errors on and
    adds a rounding (U of its result; sums of n terms n - 1 of them, of the magnitudes summed)."""

    def __init__(self, v, e=None):
        self.v, self.e = v, torch.zeros_like(v) if e is None else e

    def __add__(self, o):
        v = self.v + o.v
        return V(v, self.e + o.e + torch.where(torch.isinf(v), 0.0, U * v.abs()))      # (an infinity is not rounded)

    def __mul__(self, o):
        v = self.v * o.v
        return V(v, self.v.abs() * o.e + o.v.abs() * self.e + U * v.abs())

    def rel(self, steps):
        """Evaluated to so many half steps."""
        return V(self.v, self.e + steps * U * self.v.abs())

    def sum(self, dim, adds):
        return V(self.v.sum(dim), self.e.sum(dim) + adds * U * self.v.abs().sum(dim))

    def __getitem__(self, i):
        return V(self.v[i], self.e[i])

    def view(self, *s):
        return V(self.v.view(*s), self.e.view(*s))

    def unsqueeze(self, d):
        return V(self.v.unsqueeze(d), self.e.unsqueeze(d))


def cat(vs):
    return V(torch.cat([x.v for x in vs]), torch.cat([x.e for x in vs]))


def rounded(x, dtype):
    """(value, tolerance) of x rounded to dtype."""
    return x.v, x.e * SLACK + HALF_STEP[dtype] * (x.v.abs() + x.e) * SLACK + TINY[dtype]


def sigmoid(z):
    # an exponential to 4 half steps (its argument in two parts, the instruction's one step), a sum, an inverse of one step, a product
    g = torch.sigmoid(z.v)
    return V(g, g * (1 - g) * z.e + 9 * U * g)


def softplus(raw):
    # the exponential as above; 2 artanh(e / (2 + e)): an inverse of one step, two products and the polynomial, whose rounding is below one
    # half step of its first term; the last sum.  The smaller part of it is no more than the whole.
    s = torch.logaddexp(raw.v, torch.zeros_like(raw.v))
    return V(s, torch.sigmoid(raw.v) * raw.e + 12 * U * s + 2.0 ** -126)


def scan_terms(x, dt, a, b, c, d, z, dt_bias, rep):
    """What the recurrence is made of, per token."""
    def w(t):
        return None if t is None else V(t.double())

    raw = w(dt) if dt_bias is None else w(dt) + w(dt_bias)
    s = softplus(raw)
    xs = w(x)
    bb, cc = (V(t.double().repeat_interleave(rep, 1)) for t in (b, c))
    # the power: a log2(e) and its product with s (3 half steps of the exponent), the instruction's step; where pieces are joined, the
    # sum of 64 time steps, 18 additions deep, takes the place of the single ones
    arg = s.v[..., None] * a.double()
    decay = torch.exp(arg)
    f = V(decay, decay * (a.double().abs() * s.e[..., None] + 21 * U * arg.abs() + 2 * U) + 2.0 ** -126)
    u = s * xs
    gate = None
    if z is not None:
        zz = w(z)
        gate = zz * sigmoid(zz)
    return raw, s, xs, bb, cc, f, u, gate


def scan(x, dt, a, b, c, h0, d=None, z=None, dt_bias=None):
    """One sequence: (out, final) as V; x, dt, z [T, ch], b, c [T, groups, n], a, h0 [ch, n]."""
    rep = x.shape[1] // b.shape[1]
    _, _, xs, bb, cc, f, u, gate = scan_terms(x, dt, a, b, c, d, z, dt_bias, rep)
    h, rows = V(h0.double()), []
    add = u.unsqueeze(-1) * bb
    for t in range(x.shape[0]):
        h = f[t] * h + add[t]
        rows.append(h.unsqueeze(0))
    if not rows:
        return V(x.double()), h
    y = (cat(rows) * cc).sum(-1, a.shape[1] + 2)
    if d is not None:
        y = y + V(d.double()) * xs
    return (y if gate is None else y * gate), h


def scan_grad(dout, x, dt, a, b, c, h0, dfinal, d=None, z=None, dt_bias=None):
    """The gradients for one sequence, as V by name (token sums of a, d and dt_bias over this sequence)."""
    T, ch = x.shape
    G, n = b.shape[1], a.shape[1]
    rep = ch // G
    raw, s, xs, bb, cc, f, u, gate = scan_terms(x, dt, a, b, c, d, z, dt_bias, rep)
    add = u.unsqueeze(-1) * bb
    h, before, after = V(h0.double()), [], []
    for t in range(T):
        w = f[t] * h                # e^(s a) h_(t-1)
        h = w + add[t]
        before.append(w.unsqueeze(0))
        after.append(h.unsqueeze(0))
    g = V(dfinal.double())
    if T == 0:
        zero = V(x.double())
        return {"x": zero, "dt": zero, "z": zero, "b": V(b.double()), "c": V(c.double()), "a": V(torch.zeros_like(a.double())),
                "d": V(torch.zeros(ch, dtype=torch.float64, device=x.device)), "dt_bias": V(torch.zeros(ch, dtype=torch.float64, device=x.device)),
                "state_in": g}
    before, after = cat(before), cat(after)
    do = V(dout.double())
    dy = do if gate is None else do * gate
    into = [None] * T
    for t in range(T - 1, -1, -1):
        g = dy[t].unsqueeze(-1) * cc[t] + g
        into[t] = g.unsqueeze(0)
        g = f[t] * g
    grads = cat(into)
    adds = ch // G + 32             # a sum over channels is a tree, but no more than these deep
    out = {"c": (dy.unsqueeze(-1) * after).view(T, G, rep, n).sum(2, adds), "b": (grads * u.unsqueeze(-1)).view(T, G, rep, n).sum(2, adds)}
    if z is not None:
        y = (after * cc).sum(-1, n + 2)
        if d is not None:
            y = y + V(d.double()) * xs
        zz = V(z.double())
        sg = sigmoid(zz)
        one = V(torch.ones_like(sg.v))
        out["z"] = do * y * (sg * (zz * (one + V(-sg.v, sg.e)) + one))
    inner = (grads * bb).sum(-1, n + 2)
    out["x"] = s * inner if d is None else s * inner + dy * V(d.double())
    kk = grads * before
    up = (kk * V(a.double()).rel(3)).sum(-1, n + 4)
    ds = up + xs * inner
    slope = sigmoid(raw)
    draw = ds * slope
    out["dt"] = draw
    out["a"] = (kk * s.unsqueeze(-1)).sum(0, T + 16)
    out["d"] = (dy * xs).sum(0, T + 16)
    out["dt_bias"] = draw.sum(0, T + 16)
    out["state_in"] = g
    return out


# ---------------------------------------------------------------- e4m3

def to_e4m3(r):
    """Values (float64, numpy) within 464 to the nearest of e4m3's, halves to the even one."""
    e = np.floor(np.log2(np.maximum(np.abs(r), 2.0 ** -40)))
    step = np.exp2(np.maximum(e, -6.0) - 3.0)
    return np.rint(r / step) * step


def quantize_blocks(x, block_rows):
    """(codes as float64 values, scales float32) of x, a numpy float32 array: each step rounded to f32."""
    rows, cols = x.shape
    rb, cb = -(-rows // block_rows), -(-cols // 128)
    codes, scales = np.zeros(x.shape), np.zeros((rb, cb), np.float32)
    with np.errstate(all="ignore"):
        for i in range(rb):
            for j in range(cb):
                at = (slice(i * block_rows, (i + 1) * block_rows), slice(128 * j, 128 * j + 128))
                v = x[at]
                m = np.max(np.where(np.isnan(v), np.float32(0), np.abs(v)))
                s = np.maximum(np.float32(m) / np.float32(448), np.float32(2.0 ** -126))
                r = (v * (np.float32(1) / s)).astype(np.float32).astype(np.float64)
                codes[at], scales[i, j] = np.where(np.isnan(r), np.nan, to_e4m3(np.where(np.isnan(r), 0, r))), s
    return codes, scales


def fp8_matmul(x, sx, w, sw, bias, dtype):
    """(y, tolerance) in float64, block by block.  f32 outputs: products are exact, a block's sum of 128 at most 128 roundings of its
    magnitudes, then its factor (one rounding), a fused product and sum a block, the bias.  16-bit outputs: the matrix instruction cuts each
    product of eight neighbouring columns off, 13 bits below the exponent of the largest: seven of them by 2^-13 of that each."""
    m, k = x.shape
    n = w.shape[0]
    y = torch.zeros(m, n, dtype=torch.float64, device=x.device)
    e, mass = torch.zeros_like(y), torch.zeros_like(y)
    for c in range(0, k, 128):
        xb, wb = x[:, c:c + 128].double(), w[:, c:c + 128].double()
        f = torch.outer(sx[:, c // 128].double(), sw[:, c // 128].double().repeat_interleave(128)[:n])
        p = torch.matmul(xb, wb.T) * f
        mags = torch.matmul(xb.abs(), wb.abs().T) * f.abs()
        y = y + p
        mass = mass + mags
        e = e + 130 * U * mags + U * y.abs()
        if dtype != torch.float32:
            for g in range(0, xb.shape[1], 8):
                top = (xb[:, None, g:g + 8].abs() * wb[None, :, g:g + 8].abs()).amax(-1)
                e = e + 7 * 2.0 ** -13 * top * f.abs()
    if bias is not None:
        y = y + bias.double()
        e = e + U * y.abs()
    return y, e * SLACK + HALF_STEP[dtype] * (y.abs() + e) * SLACK + TINY[dtype]


# ---------------------------------------------------------------- sampling

ONE = 2.0 ** 42


def weights(l, temperature):
    """Whole-number weights of a row (float64 numpy), as Python ints' array (object-free: int64)."""
    l = np.where(np.isnan(l), -np.inf, l)
    top = l.max()
    with np.errstate(all="ignore"):
        w = np.where(l == top, 1.0, np.exp((l - top) / temperature))
        w = np.where(np.isneginf(l) | np.isnan(w), 0.0, w)
    return l, np.rint(w * ONE).astype(np.int64)


def kept(l, w, top_k=0, top_p=1.0, min_p=0.0):
    """The indexes that stay, in the order of their values (larger first, equal ones by index); the settings as float32."""
    order = np.lexsort((np.arange(len(l)), -l))
    order = order[w[order] > 0]
    if top_k > 0:
        order = order[:top_k]
    top_p, min_p = float(np.float32(top_p)), float(np.float32(min_p))
    if top_p < 1.0:
        sums = [0]
        for v in w[order]:
            sums.append(sums[-1] + int(v))
        need = top_p * float(sums[-1])
        order = np.array([i for j, i in enumerate(order) if j == 0 or float(sums[j]) < need], dtype=np.int64)
    if min_p > 0.0:
        order = order[w[order].astype(np.float64) >= min(min_p, 1.0) * ONE]
    return order


def draw(l, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The token of one row (numpy, any float type)."""
    l = np.asarray(l, np.float64)
    clean = np.where(np.isnan(l), -np.inf, l)
    if np.isneginf(clean.max()):
        return -1
    temperature = float(np.float32(temperature))
    if not temperature > 0:
        return int(np.argmax(clean))
    l, w = weights(l, temperature)
    keep = np.sort(kept(l, w, top_k, top_p, min_p))
    sums, total = [], 0
    for v in w[keep]:
        total += int(v)
        sums.append(total)
    u = float(np.float32(u))
    limit = (u if u > 0 else 0.0) * float(total)
    if not limit < float(total):
        limit = math.nextafter(float(total), 0.0)
    return int(next(i for i, s in zip(keep, sums) if float(s) > limit))


def draw_fast(l, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """draw by sums of whole arrays, for long rows."""
    l = np.asarray(l, np.float64)
    clean = np.where(np.isnan(l), -np.inf, l)
    if np.isneginf(clean.max()):
        return -1
    temperature, top_p, min_p, u = (float(np.float32(v)) for v in (temperature, top_p, min_p, u))
    if not temperature > 0:
        return int(np.argmax(clean))
    l, w = weights(l, temperature)
    keep = np.flatnonzero(w)
    if top_k > 0 or top_p < 1.0:
        keep = keep[np.argsort(-l[keep], kind="stable")]
        if top_k > 0:
            keep = keep[:top_k]
        if top_p < 1.0:
            sums = np.cumsum(w[keep])
            before = sums - w[keep]
            keep = keep[(before == 0) | (before.astype(np.float64) < top_p * float(sums[-1]))]
    if min_p > 0.0:
        keep = keep[w[keep].astype(np.float64) >= min(min_p, 1.0) * ONE]
    keep = np.sort(keep)
    sums = np.cumsum(w[keep])
    total = float(sums[-1])
    limit = (u if u > 0 else 0.0) * total
    if not limit < total:
        limit = math.nextafter(total, 0.0)
    return int(keep[np.argmax(sums.astype(np.float64) > limit)])
