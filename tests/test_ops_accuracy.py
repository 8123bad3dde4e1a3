"""How exact the gated delta rule over sequences is on inputs as they come, beside ops_f64's bounds on the worst ones.

The worst case of sums of hundreds of terms is hundreds of half steps, and a kernel may lose a third of its bits within it.  On random
inputs the roundings have random signs.  One f32 rounding is off by 0.41 u (u = 2^-24) in the mean square; a sum of n terms, rounded n
times at partial sums that grow to the result, by 0.41 u sqrt(n / 2) of it.  A token's row of the state comes of a sum over dk <= 128
rows of the state (3.3 u), one over the up to 64 rows of its block (2.3 u) and that block's solve (2.3 u), an output of two such sums;
the decays are good to 1 u (their logarithms are summed in 64 bits).  Together 4.8 u for the row; what was added before has decayed
together with its error, so the state's error is no larger part of it, and one more sum makes 6 u of an output.  BOUND is 8 u, on the
2-norm of a head's error over the result's.

Two limbs of bf16 where three are needed, or decays' logarithms summed in 32 bits, miss it: `emulated` is the chunk form with such
operands, on the CPU.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from redukt_amd import ops  # noqa: E402
from tests import ops_f64  # noqa: E402

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
BOUND = 8 * 2.0 ** -24
# tokens, key heads, value heads, dk, dv, decays' factor, largest strength
CASES = [(300, 1, 2, 64, 64, 1.0, 1.0), (1100, 1, 2, 128, 32, 0.01, 1.0), (500, 2, 2, 128, 64, 4.0, 1.0), (700, 1, 2, 64, 32, 0.1, 2.0)]
cases = pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-dk{c[3]}-forget{c[5]}-beta{c[6]}")


def inputs(case, dtype):
    T, hk, hv, dk, dv, forget, most = case
    r = torch.Generator().manual_seed(T)
    randn = lambda *s: torch.randn(*s, generator=r)  # noqa: E731
    q, k, v = randn(T, hk, dk), randn(T, hk, dk), randn(T, hv, dv)
    g = -forget * torch.exp(randn(1, hv) * 0.25 - 1.0) * torch.nn.functional.softplus(randn(T, hv))
    return [q.to(dtype), k.to(dtype), v.to(dtype), g, most * torch.sigmoid(randn(T, hv))], 0.3 * randn(1, hv, dk, dv)


def limbs(x, n):
    """The sum of x's first n bf16 limbs, in float32."""
    rest, total = x.clone(), torch.zeros_like(x)
    for _ in range(n):
        part = rest.to(BF16).float()
        rest, total = rest - part, total + part
    return total


def emulated(x, S, n_state, n_out, sums=torch.float64):
    """The rule in blocks of 64 tokens, in float32, normalized, with the state, its corrections and (I + A)^-1 in n_state limbs
    for the state and n_out for the outputs, and the logarithms of the decays summed in `sums`."""
    q, k, v, g, beta = x
    T, hv, dv = v.shape
    dk, rep = q.shape[2], hv // q.shape[1]
    q, k = (y.float().repeat_interleave(rep, 1) for y in (q, k))
    p, u = (1.0 / torch.sqrt((y * y).sum(-1) + 1e-6) for y in (q, k))
    p = p * dk ** -0.5
    S, out = S.clone(), torch.empty(T, hv, dv)
    for h in range(hv):
        for c in range(0, T, 64):
            e = min(c + 64, T)
            K, Q, uu, pp, b = k[c:e, h], q[c:e, h], u[c:e, h], p[c:e, h], beta[c:e, h]
            G = g[c:e, h].to(sums).cumsum(0)
            D = torch.exp((G[:, None] - G[None]).double()).tril().float()
            W = D * uu[None]
            A = (b[:, None] * uu[:, None] * W * (K @ K.T)).tril(-1)
            inv = torch.linalg.solve_triangular(torch.eye(e - c) + A, torch.eye(e - c), upper=False, unitriangular=True) * b[None]
            PT = (pp[:, None] * W * (Q @ K.T)).tril() @ inv
            eg, left = torch.exp(G.double()).float(), uu * torch.exp((G[-1] - G).double()).float()
            X = v[c:e, h].float() - (uu * eg)[:, None] * (K @ limbs(S[h], n_state))
            out[c:e, h] = (pp * eg)[:, None] * (Q @ limbs(S[h], n_out)) + limbs(PT, n_out) @ limbs(X, n_out)
            D = limbs(left[:, None] * inv, n_state) @ limbs(X, n_state)
            S[h] = eg[-1] * S[h] + K.T @ limbs(D, n_state)
    return out.to(v.dtype), S


def off(got, want, dims):
    """The 2-norm of the error of each head over the result's."""
    return float(((got.double() - want).norm(dim=dims) / want.norm(dim=dims)).max())


def exact(x, S):
    out, state, _, _ = ops_f64.rule(*x, S[0], normalize=True)
    return out, state


def rounded(out, dtype):
    """How far float64 outputs are off by their rounding to dtype alone, all heads together."""
    return float((out.to(dtype).double() - out).norm())


@cases
def test_the_bound_holds_with_three_limbs_and_notices_what_is_lost(case):
    x, S = inputs(case, F32)
    out, state = exact(x, S)
    errors = {}
    for name, args in {"three": (3, 3), "two": (2, 2), "two in the outputs": (3, 2), "sums in 32 bits": (3, 3, F32)}.items():
        o, s = emulated(x, S[0], *args)
        errors[name] = off(s, state, (1, 2)), off(o, out, (0, 2))
    assert max(errors["three"]) <= BOUND, errors
    assert min(errors["two"]) > 2 * BOUND and errors["two in the outputs"][1] > 2 * BOUND, errors
    if case[5] == 4.0:                           # (decays' sums of about 100 within a block)
        assert min(errors["sums in 32 bits"]) > BOUND, errors


@cases
def test_16_bit_outputs_of_two_limbs_are_off_by_their_rounding(case):
    """Two limbs are 16 bits: beside a rounding to 11 (0.41 * 2^-11 of the value) their error adds less than 2 % to the norm, and
    one limb's more than 10 %."""
    for dtype in (BF16, F16):
        x, S = inputs(case, dtype)
        out, _ = exact(x, S)
        two, one = (float((emulated(x, S[0], 3, n)[0].double() - out).norm()) / rounded(out, dtype) for n in (2, 1))
        assert two <= 1.02 and one > 1.1, (dtype, two, one)


# ---------------------------------------------------------------- the kernels

types = pytest.mark.parametrize("dtype", [BF16, F16, F32], ids={BF16: "bf16", F16: "f16", F32: "f32"}.get)


def as_exact(out, S, want, state, dtype, what, bound=BOUND):
    """Outputs and a state within the bound; 16-bit outputs off by their rounding alone, but for 2 %."""
    assert off(S, state, (1, 2)) <= bound, what
    if dtype == F32:
        assert off(out, want, (0, 2)) <= bound, what
    else:
        assert float((out.double() - want).norm()) <= 1.02 * rounded(want, dtype), what


@pytest.mark.gpu
@cases
@types
def test_delta_chunk_is_as_exact_as_f32_sums(case, dtype):
    """Also where a workgroup takes two column tiles and four: the same sequence many times over, with the same bits."""
    x, S = (([t.cuda() for t in y] if isinstance(y, list) else y.cuda()) for y in inputs(case, dtype))
    want, state = exact(x, S)
    T = case[0]
    after = torch.empty_like(S)
    out = ops.delta_chunk(*x, torch.tensor([0, T], dtype=torch.int32, device="cuda"), state_in=S, state_out=after, normalize=True)
    as_exact(out, after[0], want, state, dtype, "alone")
    per = case[2] * case[4] // 16
    for n in (1024 // per + 1, 2048 // per + 1):
        many = [t.repeat(n, *[1] * (t.dim() - 1)) for t in x]
        cu = torch.arange(0, n * T + 1, T, dtype=torch.int32, device="cuda")
        pool = S.repeat(n, 1, 1, 1)
        outs = ops.delta_chunk(*many, cu, state_in=pool, state_out=pool, normalize=True)
        assert (outs.view(n, *out.shape) == out).all() and (pool == after).all(), n


@pytest.mark.gpu
@types
def test_64_rows_at_most_are_as_exact(dtype):
    x, S = inputs((64, 1, 2, 64, 64, 1.0, 1.0), dtype)
    x, S = [t.cuda() for t in x], S.cuda()
    want, state = exact(x, S)
    after = torch.empty_like(S)
    out = ops.delta_chunk(*x, torch.tensor([0, 64], dtype=torch.int32, device="cuda"), state_in=S, state_out=after, normalize=True)
    as_exact(out, after[0], want, state, dtype, "64 rows")


@pytest.mark.gpu
@cases
@types
def test_delta_step_is_as_exact_token_by_token(case, dtype):
    """Token by token every decay meets the state by itself, and expf is good to 1 ulp, which is 1 u of the state below 1, perhaps with
    the same sign at every token.  An error of the state shrinks by a (1 - (2 beta - beta^2) / dk)^1/2 = r a token in the mean (a key's
    direction is one of dk), so up to u / (1 - r) of them add up: 172 u for the longest memory here, of 300 tokens by its decays.  (In
    delta_chunk the decays' logarithms are summed first, and the state meets one decay in 64 tokens.)"""
    x, S = inputs(case, dtype)
    x, S = [t.cuda() for t in x], S.cuda()
    want, state = exact(x, S)
    out = torch.cat([ops.delta_step(*(y[t:t + 1] for y in x), S, normalize=True) for t in range(case[0])])
    g, beta = (y.double().cpu() for y in x[3:])
    r = (g.exp().mean(0) * torch.sqrt(1 - (2 * beta - beta * beta).mean(0) / case[3])).max()
    as_exact(out, S[0], want, state, dtype, "steps", BOUND + 2.0 ** -24 / float(1 - r))


@pytest.mark.gpu
@types
@pytest.mark.parametrize("alike", [False, True], ids=["any keys", "alike keys"])
@pytest.mark.parametrize("dk", [64, 128])
def test_strengths_up_to_two(dk, alike, dtype):
    """I - beta k k^T does not lengthen a vector for beta |k|^2 in [0, 2], which is all that ops_f64.rule's bound takes of beta <= 1.
    Strengths of 2 itself, keys that are the same, little decay: T's entries then alternate between 2 and -2, and with 64 of them in a
    row and 64 rows their roundings sum to 0.41 u sqrt(64 * 64) * 2 = 53 u of what is added, within the bound's 2 (dk + 128) u."""
    T = 200
    x, S = inputs((T, 1, 2, dk, 64, 0.02, 2.0), dtype)
    x, S = [t.cuda() for t in x], S.cuda()
    if alike:
        x[1][:] = x[1][:1]
        x[3][:] = -1e-4
        x[4][:] = 2.0
    else:
        x[4][::3] = 2.0
        x[4][1::7] = 0.0
    want, state, tol, S_tol = ops_f64.rule(*x, S[0], normalize=True)
    after, step = torch.empty_like(S), S.clone()
    out = ops.delta_chunk(*x, torch.tensor([0, T], dtype=torch.int32, device="cuda"), state_in=S, state_out=after, normalize=True)
    steps = torch.cat([ops.delta_step(*(y[t:t + 1] for y in x), step, normalize=True) for t in range(T)])
    for o, s in ((out, after[0]), (steps, step[0])):
        assert ((o.double() - want).abs() <= tol).all() and ((s.double() - state).abs() <= S_tol).all()
