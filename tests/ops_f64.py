"""64-bit statements of the operators on caller tensors, with bounds on what f32 arithmetic and
the output's rounding may differ by."""
import numpy as np
import torch

U = 2.0 ** -24                      # half a step of f32, relative
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}      # half the smallest fp16 step


def unit(x, normalize):
    x = x.double()
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6) if normalize else x


def rule(q, k, v, g, beta, S, scale=None, normalize=False):
    """One sequence of the gated delta rule, token by token: q, k [T, hk, dk], v [T, hv, dv], g, beta [T, hv],
    S [hv, dk, dv].  Returns (out [T, hv, dv], S, out_tol, S_tol): float64 results and how far a result
    in f32, rounded to v's type, may be off.

    With |k| <= 1, beta <= 1 and a = e^g <= 1 a token takes an error in a column of S no further
    than a times its 2-norm, and adds the roundings of its own sums.  A dot product of n terms
    is off by at most n u |x||y|; one over dk columns of the state, one over the up to 64 rows
    of a block of tokens and the block's solve (64 rows again) lie behind each row that is added,
    so c = 2 (dk + 128) half steps of a (|S| + what is added) are a bound.  The outputs' sums may
    take their factors in 16 bits where the output has 16: 2^-15 of the magnitudes summed.
    """
    T, hk, dk = q.shape
    hv = v.shape[1]
    dtype = v.dtype
    q, k = (unit(x, normalize).repeat_interleave(hv // hk, 1) for x in (q, k))
    v, g, beta, S = v.double(), g.double(), beta.double(), S.double().clone()
    scale = dk ** -0.5 if scale is None else scale
    c = 2 * (dk + 128) * U
    short = 0.0 if dtype == torch.float32 else 2.0 ** -15
    err = torch.zeros_like(S[:, 0])                  # [hv, dv]: 2-norm of a column's error
    mass = S.norm(dim=1)                             # [hv, dv]: magnitudes a column was summed from
    out, tol = [], []
    for t in range(T):
        a, b = g[t].exp()[:, None], beta[t][:, None]
        norm = S.norm(dim=1)
        S = a[..., None] * S
        d = b * (v[t] - torch.matmul(k[t][:, None], S)[:, 0])
        S = S + k[t][:, :, None] * d[:, None, :]
        added = b * (v[t].abs() + a * norm)
        err = a * err + c * (a * norm + added)
        mass = a * mass + added
        o = scale * torch.matmul(q[t][:, None], S)[:, 0]
        qn = scale * q[t].norm(dim=-1)[:, None]
        out.append(o)
        tol.append(HALF_STEP[dtype] * o.abs() + TINY[dtype] + qn * (err + (c + short) * mass))
    if T == 0:
        return v.clone(), S, v.clone(), torch.zeros_like(S)
    return torch.stack(out), S, torch.stack(tol), err[:, None, :].expand_as(S) + U * S.abs()


def quantize(x):
    """(codes, scales) of rows x, a numpy float32 array: each step rounded to f32 as the recipe has it."""
    with np.errstate(all="ignore"):
        a = np.abs(x)
        m = np.max(np.where(np.isnan(a), np.float32(0), a), axis=-1, initial=np.float32(0))
        scale = np.where(m > 0, (m / np.float32(127)).astype(np.float32), np.float32(1)).astype(np.float32)
        inv = (np.float32(1) / scale).astype(np.float32)
        r = (x * inv[:, None]).astype(np.float32).astype(np.float64)
        q = np.clip(np.trunc(r + np.copysign(0.5, r)), -127, 127)
        return np.where(np.isnan(q), 0, q).astype(np.int8), scale


def matmul(x, sx, w, sw, bias, dtype):
    """(y, tol): the product in float64 (exact sums: below 2^53) and its bound: three roundings of the f32
    value (sum, product of the scales, their product), one of the bias' sum, one to dtype."""
    s = torch.matmul(x.double(), w.double().T) * sx.double()[:, None] * sw.double()
    y = s if bias is None else s + bias.double()
    return y, (4 * U * s.abs() + 2 * U * y.abs()) * 1.001 + HALF_STEP[dtype] * y.abs() * 1.001 + TINY[dtype]
