"""The operators on caller tensors (redukt_amd.ops, include/redukt_ops.h) on the GPU, against 64-bit
statements of them (tests/ops_f64.py)."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from redukt_amd import ffi, ops  # noqa: E402
from tests import ops_f64  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
NAMES = {BF16: "bf16", F16: "f16", F32: "f32"}
types = pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=NAMES.get)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rule_inputs(T, hk, hv, dk, dv, dtype, seed=0, normalize=False, forget=1.0):
    r = gen(seed)
    randn = lambda *s: torch.randn(*s, generator=r, device="cuda")  # noqa: E731
    q, k = randn(T, hk, dk), randn(T, hk, dk)
    if not normalize:
        q, k = (x / (x.norm(dim=-1, keepdim=True) * 1.01) for x in (q, k))
    v = randn(T, hv, dv)
    g = -forget * torch.exp(randn(1, hv) - 2.0) * torch.nn.functional.softplus(randn(T, hv))
    return [q.to(dtype), k.to(dtype), v.to(dtype), g, torch.sigmoid(randn(T, hv))]


def pool_of(slots, hv, dk, dv, seed=5):
    return 0.3 * torch.randn(slots, hv, dk, dv, generator=gen(seed), device="cuda")


def check(got, want, tol, what):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((off / tol.clamp(min=1e-300)).max()), float(off.max()))


def refused(call):
    with pytest.raises(ffi.BackendError) as e:
        call()
    assert e.value.result == ffi.BackendResult.INVALID_ARGUMENT


# ---------------------------------------------------------------- one token

STEP_SHAPES = [  # n, hk, hv, dk, dv, normalize
    (1, 1, 1, 64, 32, False), (1, 12, 12, 64, 64, False), (3, 2, 6, 128, 96, True), (17, 4, 4, 64, 128, True),
    (5, 1, 8, 128, 256, True), (70, 2, 2, 128, 128, False), (2, 3, 3, 64, 160, True)]


@types
@pytest.mark.parametrize("n,hk,hv,dk,dv,normalize", STEP_SHAPES)
def test_delta_step(n, hk, hv, dk, dv, normalize, dtype):
    x = rule_inputs(n, hk, hv, dk, dv, dtype, seed=n, normalize=normalize)
    pool = pool_of(n + 2, hv, dk, dv)
    slots = torch.from_numpy(np.random.default_rng(n).permutation(n + 2)[:n].astype(np.int32)).cuda()
    before = pool.clone()
    out = ops.delta_step(*x, pool, slots=slots, normalize=normalize)
    left = set(range(n + 2)) - set(slots.tolist())
    for s in left:
        assert torch.equal(pool[s], before[s])
    for i, s in enumerate(slots.tolist()):
        want, S, tol, S_tol = ops_f64.rule(*(t[i:i + 1] for t in x), before[s], normalize=normalize)
        check(out[i:i + 1], want, tol, ("out", i))
        check(pool[s], S, S_tol, ("state", i))


def test_delta_step_without_slots_and_with_a_scale():
    x = rule_inputs(4, 2, 4, 64, 64, F32)
    pool = pool_of(6, 4, 64, 64)
    before = pool.clone()
    out = torch.empty(4, 4, 64, device="cuda")
    assert ops.delta_step(*x, pool, out=out, scale=1.5) is out
    for i in range(4):
        want, S, tol, S_tol = ops_f64.rule(*(t[i:i + 1] for t in x), before[i], scale=1.5)
        check(out[i:i + 1], want, tol, i)
        check(pool[i], S, S_tol, i)
    assert torch.equal(pool[4:], before[4:])


@types
def test_delta_step_slices_of_a_projection(dtype):
    """q, k, v as slices of one projection's rows, g and beta of another's, out into a wider buffer."""
    n, hk, hv, dk, dv = 6, 2, 4, 128, 64
    x = rule_inputs(n, hk, hv, dk, dv, dtype, seed=3)
    fused = torch.cat([x[0].flatten(1), x[1].flatten(1), x[2].flatten(1)], 1)
    w = hk * dk
    q, k, v = (fused[:, :w].view(n, hk, dk), fused[:, w:2 * w].view(n, hk, dk), fused[:, 2 * w:].view(n, hv, dv))
    gates = torch.cat([x[3], x[4]], 1)
    wide = torch.full((n, hv * dv + 64), 7.0, dtype=dtype, device="cuda")
    a, b = pool_of(n, hv, dk, dv), pool_of(n, hv, dk, dv)
    out = ops.delta_step(q, k, v, gates[:, :hv], gates[:, hv:], a, out=wide[:, :hv * dv].view(n, hv, dv))
    assert torch.equal(out, ops.delta_step(*x, b)) and torch.equal(a, b)
    assert (wide[:, hv * dv:] == 7.0).all()


def test_delta_step_padded_bad_and_repeated_slots():
    n, hv, dk, dv = 7, 2, 64, 64
    x = rule_inputs(n, 2, hv, dk, dv, F32)
    for t in x:
        t[1] = float("nan")                 # a padded entry may hold anything
    pool = pool_of(4, hv, dk, dv)
    before = pool.clone()
    out = torch.full((n, hv, dv), 7.0, device="cuda")
    slots = torch.tensor([2, -1, 4, 0, 2, -7, -1], dtype=torch.int32, device="cuda")
    ops.delta_step(*x, pool, slots=slots, out=out)
    for i in (0, 3):
        s = int(slots[i])
        want, S, tol, S_tol = ops_f64.rule(*(t[i:i + 1] for t in x), before[s])
        check(out[i:i + 1], want, tol, i)
        check(pool[s], S, S_tol, i)
    for i in (1, 6):
        assert (out[i] == 7.0).all()
    for i in (2, 4, 5):
        assert out[i].isnan().all()
    assert torch.equal(pool[[1, 3]], before[[1, 3]])


def test_delta_step_extreme_decays_and_strengths():
    """A decay of e^-inf drops the state, 0 keeps it, strength 0 adds nothing, a key of zeros normalizes to zeros."""
    x = rule_inputs(4, 1, 1, 64, 64, F32, normalize=True)
    x[3][:, 0] = torch.tensor([float("-inf"), 0.0, -200.0, -0.5])
    x[4][:, 0] = torch.tensor([1.0, 0.0, 0.5, 1.0])
    x[1][3] = 0.0
    pool = pool_of(4, 1, 64, 64)
    before = pool.clone()
    out = ops.delta_step(*x, pool, normalize=True)
    for i in range(4):
        want, S, tol, S_tol = ops_f64.rule(*(t[i:i + 1] for t in x), before[i], normalize=True)
        check(out[i:i + 1], want, tol, i)
        check(pool[i], S, S_tol, i)
    assert torch.equal(pool[1], before[1])


def test_delta_step_offsets_past_32_bits():
    """A pool of more than 2^31 values: the last slot is stepped as the first one is."""
    hv, dk, dv = 32, 128, 128
    n = 2 ** 31 // (hv * dk * dv) + 2
    pool = torch.empty(n, hv, dk, dv, device="cuda")
    pool[0] = pool_of(1, hv, dk, dv)[0]
    pool[n - 1] = pool[0]
    x = [t.repeat(2, *[1] * (t.dim() - 1)) for t in rule_inputs(1, 16, hv, dk, dv, BF16)]
    out = ops.delta_step(*x, pool, slots=torch.tensor([0, n - 1], dtype=torch.int32, device="cuda"))
    assert torch.equal(out[0], out[1]) and torch.equal(pool[0], pool[n - 1])
    want, S, tol, S_tol = ops_f64.rule(*(t[:1] for t in x), pool_of(1, hv, dk, dv)[0])
    check(out[:1], want, tol, "out")
    check(pool[n - 1], S, S_tol, "state")


def test_delta_step_on_another_stream_and_captured():
    """A captured step, replayed with other eager work between, equals the eager steps on every replay."""
    x = rule_inputs(9, 2, 4, 128, 128, BF16, normalize=True)
    a, b = pool_of(9, 4, 128, 128), pool_of(9, 4, 128, 128)
    out = torch.empty(9, 4, 128, dtype=BF16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.delta_step(*x, a, out=out, normalize=True)
    torch.cuda.current_stream().wait_stream(side)
    first = ops.delta_step(*x, b, normalize=True)
    assert torch.equal(out, first) and torch.equal(a, b)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.delta_step(*x, a, out=out, normalize=True)
    for _ in range(4):
        g.replay()
        torch.cuda.synchronize()
        want = ops.delta_step(*x, b, normalize=True)
        assert torch.equal(out, want) and torch.equal(a, b)


def test_delta_step_slots_named_twice_among_many():
    """Entries far apart and neighbouring ones, each side of a thousand."""
    n = 2500
    x = rule_inputs(n, 1, 1, 64, 32, BF16)
    slots = torch.randperm(n, generator=gen(5), device="cuda").to(torch.int32)
    twice = {2499: 3, 1500: 1499, 1030: 1025, 1024: 1023, 700: 0, 2000: 64}
    lone = slots.clone()
    for late, early in twice.items():
        slots[late] = slots[early]
        lone[late] = -1
    pool = pool_of(n, 1, 64, 32)
    want_pool = pool.clone()
    got = ops.delta_step(*x, pool, slots=slots)
    want = ops.delta_step(*x, want_pool, slots=lone)
    late = torch.zeros(n, dtype=torch.bool, device="cuda")
    late[list(twice)] = True
    assert got[late].isnan().all() and torch.equal(got[~late], want[~late]) and torch.equal(pool, want_pool)


# ---------------------------------------------------------------- sequences

def sequences(lens, hk, hv, dk, dv, dtype, normalize, initial, behind=0, seed=0, forget=1.0, check_state=True):
    T = sum(lens)
    x = rule_inputs(T + behind, hk, hv, dk, dv, dtype, seed=seed, normalize=normalize, forget=forget)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    n = len(lens)
    slots = torch.from_numpy(np.random.default_rng(seed).permutation(n + 2)[:n].astype(np.int32)).cuda()
    before = pool_of(n + 2, hv, dk, dv) if initial else None
    after = torch.full((n + 2, hv, dk, dv), 7.0, device="cuda")
    out = torch.full((T + behind, hv, dv), 7.0, dtype=dtype, device="cuda")
    ops.delta_chunk(*x, cu, state_in=before, state_out=after, slots=slots, out=out, normalize=normalize)
    start = 0
    for i, (length, s) in enumerate(zip(lens, slots.tolist())):
        S0 = before[s] if initial else torch.zeros(hv, dk, dv, device="cuda")
        rows = slice(start, start + length)
        want, S, tol, S_tol = ops_f64.rule(*(t[rows] for t in x), S0, normalize=normalize)
        check(out[rows], want, tol, ("out", i))
        check(after[s], S, S_tol, ("state", i))
        start += length
    assert (out[T:] == 7.0).all()
    for s in set(range(n + 2)) - set(slots.tolist()):
        assert (after[s] == 7.0).all()


@types
@pytest.mark.parametrize("lens", [[1], [2], [15], [16], [17], [63], [64], [65], [128], [200], [1, 64, 0, 3, 129, 0]],
                         ids=lambda v: "-".join(map(str, v)))
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128)])
def test_delta_chunk_lengths(lens, dk, dv, dtype):
    sequences(lens, 2, 4, dk, dv, dtype, normalize=dk == 128, initial=True, behind=3, seed=len(lens) + lens[0])


@types
@pytest.mark.parametrize("lens", [[64], [30, 0, 34], [1] * 16, [5, 0, 0, 50, 3]], ids=lambda v: "-".join(map(str, v)))
@pytest.mark.parametrize("dk,dv,hk,hv", [(64, 64, 2, 2), (128, 160, 1, 3), (128, 256, 1, 16)])
def test_delta_chunk_of_64_rows_at_most(dk, dv, hk, hv, lens, dtype):
    """Few rows in all, with few column tiles and with many."""
    sequences(lens, hk, hv, dk, dv, dtype, normalize=hk == 1, initial=True, seed=hv)


@types
@pytest.mark.parametrize("which", ["v", "k", "g", "beta"])
def test_delta_chunk_of_50_rows_what_is_not_finite(which, dtype):
    x = rule_inputs(50, 2, 2, 64, 64, dtype, seed=2, normalize=True)
    cu = torch.tensor([0, 20, 50], dtype=torch.int32, device="cuda")
    S = torch.zeros(2, 2, 64, 64, device="cuda")
    want = ops.delta_chunk(*x, cu, state_out=S, normalize=True)
    y = [t.clone() for t in x]
    y[{"v": 2, "k": 1, "g": 3, "beta": 4}[which]][33, 1] = float("nan")
    S2 = torch.zeros_like(S)
    got = ops.delta_chunk(*y, cu, state_out=S2, normalize=True)
    bad = torch.zeros(50, 2, 64, dtype=torch.bool, device="cuda")
    bad[33:, 1] = True
    assert torch.equal(got[~bad], want[~bad]) and not torch.isfinite(got[bad]).any()
    assert torch.equal(S2[0], S[0]) and torch.equal(S2[1, 0], S[1, 0]) and not torch.isfinite(S2[1, 1]).any()


@types
@pytest.mark.parametrize("hk,hv,dk,dv", [(1, 1, 64, 32), (3, 3, 64, 96), (1, 4, 128, 64), (2, 2, 128, 256), (4, 12, 64, 160)])
def test_delta_chunk_heads(hk, hv, dk, dv, dtype):
    sequences([70, 1, 130], hk, hv, dk, dv, dtype, normalize=True, initial=False, seed=hv)


@types
@pytest.mark.parametrize("n", [12, 23, 66])
@pytest.mark.parametrize("dk,dv", [(64, 128), (128, 160)])
def test_delta_chunk_many_sequences(dk, dv, n, dtype):
    """Enough sequences that a workgroup takes several column tiles (two, four), and several heads of the preparation, in the
    order of their lengths and not: the same bits as each sequence alone, and the rule's values."""
    hk, hv = 6, 12
    lens = [(7 * i) % 61 + 70 * (i % 9 == 0) for i in range(n)]
    T = sum(lens)
    x = rule_inputs(T, hk, hv, dk, dv, dtype, seed=6, normalize=True)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    at = cu.tolist()
    before = pool_of(n, hv, dk, dv)
    after = torch.empty_like(before)
    out = ops.delta_chunk(*x, cu, state_in=before, state_out=after, normalize=True)
    for i in (0, 1, 9, n // 2, n - 1):
        rows = slice(at[i], at[i + 1])
        want, S, tol, S_tol = ops_f64.rule(*(t[rows] for t in x), before[i], normalize=True)
        check(out[rows], want, tol, ("out", i))
        check(after[i], S, S_tol, ("state", i))
    for i in range(n):
        rows = slice(at[i], at[i + 1])
        one = torch.empty_like(before[:1])
        alone = ops.delta_chunk(*(t[rows] for t in x), torch.tensor([0, lens[i]], dtype=torch.int32, device="cuda"),
                                state_in=before[i:i + 1], state_out=one, normalize=True)
        assert torch.equal(out[rows], alone) and torch.equal(after[i], one[0]), i


@pytest.mark.parametrize("dtype,forget", [(BF16, 1.0), (F32, 1.0), (F32, 0.01), (BF16, 30.0)])
def test_delta_chunk_long(dtype, forget):
    """Long memories and short ones (forget: the decays' factor) over some thousand tokens."""
    sequences([2111], 1, 2, 128, 64, dtype, normalize=True, initial=True, seed=9, forget=forget)


@types
def test_delta_chunk_alike_keys(dtype):
    """The same key at every token, strength 1, little decay: the block's solve is as far from the identity as it gets."""
    T, dk, dv = 150, 64, 64
    x = rule_inputs(T, 1, 1, dk, dv, dtype, normalize=True)
    x[1][:] = x[1][:1]
    x[3][:] = -1e-4
    x[4][:] = 1.0
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    S = torch.zeros(1, 1, dk, dv, device="cuda")
    out = ops.delta_chunk(*x, cu, state_out=S, normalize=True)
    want, S64, tol, S_tol = ops_f64.rule(*x, S[0] * 0, normalize=True)
    check(out, want, tol, "out")
    check(S[0], S64, S_tol, "state")


@types
def test_delta_chunk_extreme_decays(dtype):
    """Decays of e^-inf and of e^-90 within a block, beside tokens that keep everything."""
    T, dk, dv = 140, 64, 64
    x = rule_inputs(T, 2, 2, dk, dv, dtype)
    x[3][:] = 0.0
    x[3][5, 0] = float("-inf")
    x[3][64, 0] = float("-inf")
    x[3][70:100, 1] = -90.0
    x[3][101, 1] = -3.0
    x[4][20:30] = 0.0
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    before = pool_of(1, 2, dk, dv)
    after = torch.empty_like(before)
    out = ops.delta_chunk(*x, cu, state_in=before, state_out=after)
    want, S, tol, S_tol = ops_f64.rule(*x, before[0])
    check(out, want, tol, "out")
    check(after[0], S, S_tol, "state")


def test_delta_chunk_of_values_of_many_sizes():
    """Values from 1e-20 to 1e20 in neighbouring columns: columns do not meet."""
    T, dk, dv = 100, 64, 64
    x = rule_inputs(T, 1, 1, dk, dv, BF16, normalize=True)
    size = torch.logspace(-20, 20, dv, device="cuda")
    x[2] = (x[2].float() * size).to(BF16)
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    S = torch.zeros(1, 1, dk, dv, device="cuda")
    out = ops.delta_chunk(*x, cu, state_out=S, normalize=True)
    want, S64, tol, S_tol = ops_f64.rule(*x, S[0] * 0, normalize=True)
    check(out, want, tol, "out")
    check(S[0], S64, S_tol, "state")


@types
@pytest.mark.parametrize("which", ["v", "k", "q", "g", "beta", "g_inf", "state"])
@pytest.mark.parametrize("at", [0, 29, 64, 99])
def test_delta_chunk_what_is_not_finite_reaches_no_earlier_token(which, at, dtype):
    """A value that is not finite at one token leaves every earlier token's output as it was, and other columns, heads
    and sequences where the rule does not carry it to them."""
    lens, dk, dv = [130, 70], 64, 64
    x = rule_inputs(200, 2, 2, dk, dv, dtype, seed=2, normalize=True)
    cu = torch.tensor([0, 130, 200], dtype=torch.int32, device="cuda")
    before = pool_of(2, 2, dk, dv)
    S = torch.empty_like(before)
    want = ops.delta_chunk(*x, cu, state_in=before, state_out=S, normalize=True)
    y, start = [t.clone() for t in x], before.clone()
    cols = slice(None)
    if which == "v":
        y[2][at, 1, 5] = float("nan")
        cols = slice(5, 6)
    elif which == "state":
        start[0, 1, 3, 5] = float("inf")
        cols, at = slice(5, 6), 0
    elif which == "g_inf":
        y[3][at, 1] = float("inf")
    else:
        y[{"q": 0, "k": 1, "g": 3, "beta": 4}[which]][at, 1] = float("nan")
    S2 = torch.empty_like(before)
    got = ops.delta_chunk(*y, cu, state_in=start, state_out=S2, normalize=True)
    bad = torch.zeros(200, 2, dv, dtype=torch.bool, device="cuda")
    if which == "q":
        bad[at, 1] = True
    else:
        bad[at:130, 1, cols] = True
        assert S2[0, 1, :, cols].isnan().all()
        S2[0, 1, :, cols] = S[0, 1, :, cols]
    assert got[bad].isnan().all() and torch.equal(got[~bad], want[~bad])
    assert torch.equal(S2, S)


def test_delta_chunk_in_place_shared_and_bad_slots():
    hv, dk, dv = 2, 64, 64
    lens = [40, 70, 3, 5, 9]
    x = rule_inputs(sum(lens), 2, hv, dk, dv, F32)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    at = cu.tolist()
    pool = pool_of(4, hv, dk, dv)
    before = pool.clone()
    slots = torch.tensor([1, -1, 1, 9, 3], dtype=torch.int32, device="cuda")
    out = torch.full((sum(lens), hv, dv), 7.0, device="cuda")
    ops.delta_chunk(*x, cu, state_in=pool, state_out=pool, slots=slots, out=out)
    for i in (0, 4):
        rows = slice(at[i], at[i + 1])
        want, S, tol, S_tol = ops_f64.rule(*(t[rows] for t in x), before[int(slots[i])])
        check(out[rows], want, tol, i)
        check(pool[int(slots[i])], S, S_tol, i)
    assert (out[at[1]:at[2]] == 7.0).all()
    for i in (2, 3):
        assert out[at[i]:at[i + 1]].isnan().all()
    assert torch.equal(pool[[0, 2]], before[[0, 2]])
    # without final states several sequences may start from one slot
    slots = torch.tensor([1, 0, 1, 1, 3], dtype=torch.int32, device="cuda")
    out = ops.delta_chunk(*x, cu, state_in=before, slots=slots)
    for i, s in enumerate(slots.tolist()):
        rows = slice(at[i], at[i + 1])
        want, _, tol, _ = ops_f64.rule(*(t[rows] for t in x), before[s])
        check(out[rows], want, tol, i)
    # and without any state there are no slots
    out = ops.delta_chunk(*x, cu)
    want, _, tol, _ = ops_f64.rule(*(t[:40] for t in x), before[0] * 0)
    check(out[:40], want, tol, "no state")


def test_delta_chunk_no_rows():
    """Sequences without rows hand their first state on (zeros where there is none)."""
    x = rule_inputs(0, 2, 2, 64, 64, BF16)
    cu = torch.zeros(4, dtype=torch.int32, device="cuda")
    before, after = pool_of(3, 2, 64, 64), pool_of(3, 2, 64, 64, seed=8)
    assert ops.delta_chunk(*x, cu, state_in=before, state_out=after).shape == (0, 2, 64)
    assert torch.equal(before, after)
    ops.delta_chunk(*x, cu, state_out=after)
    assert (after == 0).all()
    assert ops.delta_chunk(*x, cu[:1]).shape == (0, 2, 64)


def test_delta_chunk_bad_lengths_stay_within_the_arrays():
    """Values of cu_seqlens outside the rows, or decreasing ones, reach nothing outside the arrays."""
    x = rule_inputs(100, 1, 1, 64, 64, BF16)
    wide = torch.full((300, 1, 64), 7.0, dtype=BF16, device="cuda")
    cu = torch.tensor([-50, 30, 20, 90, 10 ** 9], dtype=torch.int32, device="cuda")
    ops.delta_chunk(*x, cu, out=wide[100:200])
    assert (wide[:100] == 7.0).all() and (wide[200:] == 7.0).all()


def test_delta_chunk_captured_twice_with_a_workspace_each():
    lens = [130, 5, 77]
    x = rule_inputs(sum(lens), 2, 4, 128, 128, BF16, normalize=True)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    before = pool_of(3, 4, 128, 128)
    graphs = []
    for _ in range(2):
        S, out = before.clone(), torch.empty(sum(lens), 4, 128, dtype=BF16, device="cuda")
        need = ops.delta_chunk_workspace(sum(lens), 3, 2, 4, 128, 128, BF16)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.delta_chunk(*x, cu, state_in=S, state_out=S, out=out, normalize=True, workspace=ws)
        graphs.append((g, S, out, ws))
    S = before.clone()
    for _ in range(3):
        for g, *_ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = ops.delta_chunk(*x, cu, state_in=S, state_out=S, normalize=True)
        for _, s, out, _ in graphs:
            assert torch.equal(out, want) and torch.equal(s, S)


def test_delta_chunk_replayed_with_other_lengths_and_slots():
    """A captured call reads the lengths and slots, like everything else, when it is replayed."""
    T, n = 300, 5
    x = rule_inputs(T, 2, 4, 64, 64, BF16, normalize=True)
    cu, slots = torch.zeros(n + 1, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    pool, eager = pool_of(8, 4, 64, 64), pool_of(8, 4, 64, 64)
    out = torch.full((T, 4, 64), 7.0, dtype=BF16, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.delta_chunk(*x, cu, state_in=pool, state_out=pool, slots=slots, out=out, normalize=True)
    for at, to in [([0, 300, 300, 300, 300, 300], [0, 1, 2, 3, 4]), ([7, 20, 21, 150, 150, 299], [5, -1, 0, 7, 5]),
                   ([0, 0, 64, 128, 129, 300], [4, 3, 2, 1, 0]), ([10, 20, 30, 40, 50, 60], [-1, -1, -1, 8, -2])]:
        cu.copy_(torch.tensor(at, dtype=torch.int32))
        slots.copy_(torch.tensor(to, dtype=torch.int32))
        out.fill_(7.0)
        want = torch.full_like(out, 7.0)
        g.replay()
        torch.cuda.synchronize()
        ops.delta_chunk(*x, cu, state_in=eager, state_out=eager, slots=slots, out=want, normalize=True)
        assert torch.equal(out.nan_to_num(9.0), want.nan_to_num(9.0)) and torch.equal(pool, eager)
        assert (want[:at[0]] == 7.0).all() and (want[at[-1]:] == 7.0).all() and not (want[:at[0]] != want[:at[0]]).any()


@types
def test_delta_chunk_slices_of_a_projection(dtype):
    n, hk, hv, dk, dv = 200, 2, 4, 128, 64
    x = rule_inputs(n, hk, hv, dk, dv, dtype, seed=3, normalize=True)
    fused = torch.cat([torch.full((n, 8), float("nan"), dtype=dtype, device="cuda")] + [t.flatten(1) for t in x[:3]], 1)
    w, o = hk * dk, 8
    q, k, v = (fused[:, o:o + w].view(n, hk, dk), fused[:, o + w:o + 2 * w].view(n, hk, dk), fused[:, o + 2 * w:].view(n, hv, dv))
    gates = torch.cat([x[3], x[4]], 1)
    wide = torch.full((n, hv * dv + 64), 7.0, dtype=dtype, device="cuda")
    cu = torch.tensor([0, 3, 131, n], dtype=torch.int32, device="cuda")
    a, b = torch.empty(3, hv, dk, dv, device="cuda"), torch.empty(3, hv, dk, dv, device="cuda")
    out = ops.delta_chunk(q, k, v, gates[:, :hv], gates[:, hv:], cu, state_out=a, out=wide[:, :hv * dv].view(n, hv, dv), normalize=True)
    assert torch.equal(out, ops.delta_chunk(*x, cu, state_out=b, normalize=True)) and torch.equal(a, b)
    assert (wide[:, hv * dv:] == 7.0).all()


def test_delta_chunk_offsets_past_32_bits():
    """Rows and states beyond 2^32 bytes: the last sequence of many rows is the same as alone."""
    hk, hv, dk, dv, n = 1, 64, 64, 256, 140000
    x = rule_inputs(100, hk, hv, dk, dv, BF16, normalize=True)
    wide = [torch.zeros(n, *t.shape[1:], dtype=t.dtype, device="cuda") for t in x]
    for t, part in zip(wide, x):
        t[n - 100:] = part
    slots = 2 ** 31 // (hv * dk * dv) + 2
    pool, one = torch.empty(slots, hv, dk, dv, device="cuda"), pool_of(1, hv, dk, dv)
    pool[slots - 1] = one[0]
    cu = torch.tensor([n - 100, n], dtype=torch.int32, device="cuda")
    out = ops.delta_chunk(*wide, cu, state_in=pool, state_out=pool, slots=torch.tensor([slots - 1], dtype=torch.int32, device="cuda"), normalize=True)
    want = ops.delta_chunk(*x, torch.tensor([0, 100], dtype=torch.int32, device="cuda"), state_in=one, state_out=one, normalize=True)
    assert torch.equal(out[n - 100:], want) and torch.equal(pool[slots - 1], one[0])


def test_the_most_entries_and_sequences():
    n = 65536
    x = rule_inputs(n, 1, 1, 64, 32, BF16)
    pool = pool_of(n, 1, 64, 32)
    before = pool.clone()
    out = ops.delta_step(*x, pool)
    S = before.clone()
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    chunk = ops.delta_chunk(*x, cu, state_in=S, state_out=S)
    at = [0, 1, 40000, n - 1]
    for i in at:
        want, S64, tol, S_tol = ops_f64.rule(*(t[i:i + 1] for t in x), before[i])
        check(out[i:i + 1], want, tol, i)
        check(chunk[i:i + 1], want, tol, i)
        check(pool[i], S64, S_tol, i)
        check(S[i], S64, S_tol, i)
    more = [torch.cat([t, t[:1]]) for t in x]
    refused(lambda: ops.delta_step(*more, torch.empty(n + 1, 1, 64, 32, device="cuda")))
    refused(lambda: ops.delta_chunk(*more, torch.arange(n + 2, dtype=torch.int32, device="cuda")))


def test_two_streams_at_once():
    """Calls on two streams with nothing in common, workspaces of their own, several times over."""
    sides = [torch.cuda.Stream() for _ in range(2)]
    jobs = []
    for k in range(2):
        lens = [700 + 300 * k, 64, 130]
        x = rule_inputs(sum(lens), 4, 8, 128, 128, BF16, seed=k, normalize=True)
        cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
        codes = product(300, 280, 320, seed=k)
        S = torch.empty(3, 8, 128, 128, device="cuda")
        jobs.append((x, cu, S, codes, ops.delta_chunk(*x, cu, state_out=S, normalize=True), S.clone(), ops.int8_matmul(*codes)))
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for side, (x, cu, S, codes, *_) in zip(sides, jobs):
            with torch.cuda.stream(side):
                S.zero_()
                got.append((ops.delta_chunk(*x, cu, state_out=S, normalize=True), ops.int8_matmul(*codes)))
        torch.cuda.synchronize()
        for (out, y), (_, _, S, _, want, S_want, y_want) in zip(got, jobs):
            assert torch.equal(out, want) and torch.equal(S, S_want) and torch.equal(y, y_want)


@types
def test_a_sequence_alone_is_the_sequence_in_a_batch(dtype):
    """A sequence's bits do not depend on what else the call holds."""
    lens = [33, 190, 64]
    x = rule_inputs(sum(lens), 2, 4, 64, 64, dtype, seed=4)
    cu = torch.tensor([0, 33, 223, 287], dtype=torch.int32, device="cuda")
    S = torch.zeros(3, 4, 64, 64, device="cuda")
    out = ops.delta_chunk(*x, cu, state_out=S)
    one = torch.zeros(1, 4, 64, 64, device="cuda")
    alone = ops.delta_chunk(*(t[33:223] for t in x), torch.tensor([0, 190], dtype=torch.int32, device="cuda"), state_out=one)
    assert torch.equal(out[33:223], alone) and torch.equal(S[1], one[0])


def test_tensors_that_do_not_belong_together_are_refused():
    q, k, v, g, beta = x = rule_inputs(4, 2, 4, 64, 64, BF16)
    pool = pool_of(6, 4, 64, 64)
    before = pool.clone()
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    slots = torch.zeros(4, dtype=torch.int32, device="cuda")
    sixth = torch.zeros(4, 6, 64, dtype=BF16, device="cuda")
    bad = [(q.cpu(), k, v, g, beta), (q.float(), k, v, g, beta), (q, k[:3], v, g, beta), (q, k, v.float(), g, beta), (q, k, v[0], g, beta),
           (q, k, v, g.double(), beta), (q, k, v, g[:, :3], beta), (q, k, v, g, beta.cpu()), (q, k, None, g, beta), (q.int(), k, v, g, beta),
           (q, k, v.transpose(1, 2), g, beta), (q[..., ::2], k[..., ::2], v, g, beta), (q, k, sixth[:, :5], torch.zeros(4, 5, device="cuda"), torch.zeros(4, 5, device="cuda")),
           (q[:1].expand(4, 2, 64), k, v, g, beta)]
    for y in bad:
        refused(lambda: ops.delta_step(*y, pool))
        refused(lambda: ops.delta_chunk(*y, cu))
    for states in (pool.half(), pool[:3], pool[:, :3], pool.transpose(2, 3), pool.cpu(), None):
        refused(lambda: ops.delta_step(*x, states))
        if states is not None:
            refused(lambda: ops.delta_chunk(*x, torch.zeros(5, dtype=torch.int32, device="cuda"), state_out=states))
    for s in (slots.long(), slots[:3], slots.cpu(), slots[None]):
        refused(lambda: ops.delta_step(*x, pool, slots=s))
    refused(lambda: ops.delta_step(*x, pool, out=torch.empty(4, 4, 64, device="cuda")))
    refused(lambda: ops.delta_chunk(*x, cu.long()))
    refused(lambda: ops.delta_chunk(*x, cu[:0]))
    refused(lambda: ops.delta_chunk(*x, cu, slots=slots[:1]))                                     # slots of no pool
    refused(lambda: ops.delta_chunk(*x, cu, state_in=pool, state_out=pool[:3]))
    both = torch.zeros(7, 4, 64, 64, device="cuda")
    refused(lambda: ops.delta_chunk(*x, cu, state_in=both[:6], state_out=both[1:]))                # overlap in part
    need = ops.delta_chunk_workspace(4, 1, 2, 4, 64, 64, BF16)
    refused(lambda: ops.delta_chunk(*x, cu, workspace=torch.empty(need - 1, dtype=torch.uint8, device="cuda")))
    refused(lambda: ops.delta_chunk(*x, cu, workspace=torch.empty(need + 16, dtype=torch.uint8, device="cuda")[1:]))
    codes, s = ops.quantize_rows(q.flatten(1))
    w, sw = codes, s
    refused(lambda: ops.quantize_rows(q))
    refused(lambda: ops.quantize_rows(codes))
    refused(lambda: ops.quantize_rows(q.flatten(1), codes=codes[:, :5]))
    refused(lambda: ops.quantize_rows(q.flatten(1).t()))
    for y in [(codes.int(), s, w, sw), (codes, s[:3], w, sw), (codes, s, w[:, :5], sw), (codes, s.double(), w, sw), (codes, s, w, sw.cpu()),
              (codes[:, ::2], s, w[:, ::2], sw), (codes[0], s, w, sw)]:
        refused(lambda: ops.int8_matmul(*y))
    refused(lambda: ops.int8_matmul(codes, s, w, sw, bias=sw[:2]))
    refused(lambda: ops.int8_matmul(codes, s, w, sw, dtype=torch.float64))
    refused(lambda: ops.int8_matmul(codes, s, w, sw, out=torch.empty(4, 5, device="cuda")))
    assert torch.equal(pool, before)


def test_gradients_and_allocations_on_other_streams_are_refused():
    q, k, v, g, beta = x = rule_inputs(4, 2, 4, 64, 64, BF16)
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    codes, s = ops.quantize_rows(q.flatten(1))
    for i in range(5):
        y = list(x)
        y[i] = y[i].clone().requires_grad_()
        refused(lambda: ops.delta_step(*y, pool_of(4, 4, 64, 64)))
        refused(lambda: ops.delta_chunk(*y, cu))
        with torch.no_grad():
            ops.delta_step(*y, pool_of(4, 4, 64, 64))
    refused(lambda: ops.quantize_rows(q.flatten(1).clone().requires_grad_()))
    refused(lambda: ops.int8_matmul(codes, s, codes, s.clone().requires_grad_()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    work = torch.empty(ops.delta_chunk_workspace(4, 1, 2, 4, 64, 64, BF16), dtype=torch.uint8, device="cuda")
    raw, out = side.cuda_stream, torch.empty_like(v)
    refused(lambda: ops.delta_step(*x, pool_of(4, 4, 64, 64), stream=raw))
    refused(lambda: ops.delta_chunk(*x, cu, out=out, stream=raw))
    refused(lambda: ops.delta_chunk(*x, cu, workspace=work, stream=raw))
    refused(lambda: ops.quantize_rows(q.flatten(1), codes=codes, stream=raw))
    refused(lambda: ops.int8_matmul(codes, s, codes, s, stream=raw))
    want = ops.delta_chunk(*x, cu)
    ops.delta_chunk(*x, cu, out=out, workspace=work, stream=raw)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    assert torch.equal(ops.delta_chunk(*x, cu, stream=torch.cuda.current_stream().cuda_stream), want)


def test_sizes_whose_launch_does_not_fit_are_refused():
    q, k, v, g, beta = rule_inputs(1, 1, 4096, 64, 256, BF16)
    a, out, _ = ops._rows("", q, k, v, g, beta, None, None, False)
    a.rows, a.q_stride, a.k_stride, a.v_stride, a.out_stride = 65536, 64, 64, 1 << 20, 1 << 20
    out.zero_()
    L, here, no = ops._load(), torch.cuda.current_stream().cuda_stream, int(ffi.BackendResult.INVALID_ARGUMENT)
    assert L.redukt_op_delta_step(ctypes.byref(a), g.data_ptr(), 65536, None, here) == no
    cu = torch.zeros(2, dtype=torch.int32, device="cuda")
    work = torch.empty(16, dtype=torch.uint8, device="cuda")
    assert L.redukt_op_delta_chunk(ctypes.byref(a), cu.data_ptr(), 65536, None, None, 0, None, work.data_ptr(), 1 << 60, here) == no
    torch.cuda.synchronize()
    assert not out.any()


# ---------------------------------------------------------------- codes

@types
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 768), (3, 7), (5, 64), (2, 1000), (4, 4096), (3, 4097), (2, 20000), (300, 200)])
def test_quantize_rows(rows, cols, dtype):
    x = torch.randn(rows, cols, generator=gen(cols), device="cuda")
    x *= torch.exp(3 * torch.randn(rows, 1, generator=gen(rows), device="cuda"))
    x = x.to(dtype)
    codes, scales = ops.quantize_rows(x)
    want, s = ops_f64.quantize(x.float().cpu().numpy())
    assert np.array_equal(scales.cpu().numpy().view(np.uint32), s.view(np.uint32))
    assert np.array_equal(codes.cpu().numpy(), want)


@types
def test_quantize_rows_of_special_values(dtype):
    big = torch.finfo(dtype).max
    rows = [[0.0] * 9, [float("nan")] * 9, [1.0, -1.0, float("nan"), 0.5, 0.25, -0.25, 0.0, 2.0, -2.0],
            [float("inf"), 1.0, -1.0, 0.0, -float("inf"), 2.0, 3.0, 4.0, 5.0], [big, -big, big / 2, 0, 1, 2, 3, 4, 5],
            [127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 63.5, -63.5], [1e-7, 5e-8, -1e-7, 0, 0, 0, 0, 0, 0]]
    x = torch.tensor(rows, device="cuda").to(dtype)
    codes, scales = ops.quantize_rows(x)
    want, s = ops_f64.quantize(x.float().cpu().numpy())
    assert np.array_equal(scales.cpu().numpy(), s) and np.array_equal(codes.cpu().numpy(), want)


@types
@pytest.mark.parametrize("off,pad", [(0, 1), (1, 0), (3, 5), (8, 8)])
def test_quantize_rows_strided_and_unaligned(off, pad, dtype):
    rows, cols = 5, 321
    wide = torch.randn(rows, off + cols + pad, generator=gen(1), device="cuda").to(dtype)
    x = wide[:, off:off + cols]
    codes = torch.full((rows, cols + off + pad), 99, dtype=torch.int8, device="cuda")
    _, scales = ops.quantize_rows(x, codes=codes[:, off:off + cols])
    want, s = ops_f64.quantize(x.float().cpu().numpy())
    assert np.array_equal(codes[:, off:off + cols].cpu().numpy(), want) and np.array_equal(scales.cpu().numpy(), s)
    assert (codes[:, :off] == 99).all() and (codes[:, off + cols:] == 99).all()


@pytest.mark.parametrize("rows, cols", [((1 << 26) + 5, 1), ((1 << 24) + 5, 260)])
def test_more_rows_than_one_dimension_of_a_launch(rows, cols):
    x = torch.zeros(rows, cols, dtype=torch.float16, device="cuda")
    at = torch.tensor([0, 1, (1 << 22) - 1, 1 << 22, (1 << 24) + 1, rows - 1], device="cuda")
    x[at, cols - 1] = torch.tensor([1.0, -2.0, 3.0, -4.0, 5.0, -6.0], dtype=torch.float16, device="cuda")
    codes, s = ops.quantize_rows(x)
    want, ws = ops.quantize_rows(x[at])
    assert torch.equal(codes[at], want) and torch.equal(s[at], ws)
    assert int(codes.count_nonzero()) == 6 and int((s == 1.0).sum()) == rows - 6


# ---------------------------------------------------------------- product

def product(m, n, k, seed=0):
    r = gen(seed)
    code = lambda a, b: torch.randint(-128, 128, (a, b), generator=r, device="cuda", dtype=torch.int8)  # noqa: E731
    return (code(m, k), torch.exp(torch.randn(m, generator=r, device="cuda")) / 128, code(n, k),
            torch.exp(torch.randn(n, generator=r, device="cuda")) / 128, torch.randn(n, generator=r, device="cuda"))


@types
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 16, 16), (1, 1000, 768), (2, 33, 48), (7, 300, 64), (16, 16, 1536), (17, 129, 80),
                                   (33, 64, 128), (64, 250, 192), (65, 512, 256), (100, 100, 100), (128, 128, 64), (200, 300, 336),
                                   (257, 255, 512), (130, 700, 17), (3, 5, 4099), (1, 40, 16384), (600, 520, 1024), (8, 8200, 256), (3, 8200, 144), (1800, 1800, 160), (2200, 2200, 96),
                                   (4100, 4100, 80), (20, 96, 1040), (900, 1100, 400)])
def test_int8_matmul(m, n, k, dtype):
    x, sx, w, sw, bias = product(m, n, k, seed=m + n)
    for b in (None, bias):
        y = ops.int8_matmul(x, sx, w, sw, bias=b, dtype=dtype)
        check(y, *ops_f64.matmul(x, sx, w, sw, b, dtype), "y")


def test_int8_matmul_without_columns():
    x, sx, w, sw, bias = product(5, 7, 0)
    assert torch.equal(ops.int8_matmul(x, sx, w, sw, bias=bias, dtype=F32), bias.expand(5, 7))
    assert (ops.int8_matmul(x, sx, w, sw, dtype=F32) == 0).all()
    assert ops.int8_matmul(x[:0], sx[:0], w, sw).shape == (0, 7)


def test_int8_matmul_of_the_largest_codes():
    """Sums next to the end of 32 bits: -128 times -128 over the most columns."""
    k = 131000
    x = torch.full((2, k), -128, dtype=torch.int8, device="cuda")
    w = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
    one = torch.ones(3, device="cuda")
    y = ops.int8_matmul(x, one[:2], w, one, dtype=F32)
    check(y, *ops_f64.matmul(x, one[:2], w, one, None, F32), "y")
    refused(lambda: ops.int8_matmul(x.repeat(1, 2), one[:2], w.repeat(1, 2), one))


@types
@pytest.mark.parametrize("m,n,k", [(4, 70, 64), (100, 140, 128), (300, 280, 320)])
@pytest.mark.parametrize("off,pad", [(0, 16), (16, 0), (1, 0), (0, 3)])
def test_int8_matmul_strided_and_unaligned(m, n, k, off, pad, dtype):
    x, sx, w, sw, bias = product(m, n, k)
    wide = lambda t: torch.cat([torch.full((t.shape[0], off), 77, dtype=torch.int8, device="cuda"), t,  # noqa: E731
                                torch.full((t.shape[0], pad), 77, dtype=torch.int8, device="cuda")], 1)[:, off:off + k]
    out = torch.full((m, off + n + pad), 7.0, dtype=dtype, device="cuda")
    ops.int8_matmul(wide(x), sx, wide(w), sw, bias=bias, out=out[:, off:off + n])
    check(out[:, off:off + n], *ops_f64.matmul(x, sx, w, sw, bias, dtype), "y")
    assert (out[:, :off] == 7.0).all() and (out[:, off + n:] == 7.0).all()


@pytest.mark.parametrize("m,n,of", [(45000, 50280, "out"), (4200, 300, "x"), (3, 1100, "w"), (300, 1100, "w")])
def test_int8_matmul_offsets_past_32_bits(m, n, of):
    x, sx, w, sw, bias = product(m, n, 64)
    wx, ww = x, w
    if of == "x":
        wx = torch.empty(m, 1 << 20, dtype=torch.int8, device="cuda")[:, :64].copy_(x)
    if of == "w":
        ww = torch.empty(n, 1 << 22, dtype=torch.int8, device="cuda")[:, :64].copy_(w)
    got = ops.int8_matmul(wx, sx, ww, sw, bias=bias)
    for rows in (slice(0, 3), slice(m - 3, m)):
        assert torch.equal(got[rows], ops.int8_matmul(x[rows], sx[rows], w, sw, bias=bias))


@pytest.mark.parametrize("m,n,k", [(3, 1000, 768), (100, 500, 512), (700, 600, 256)])
def test_int8_matmul_captured(m, n, k):
    x, sx, w, sw, _ = product(m, n, k)
    out = torch.empty(m, n, dtype=F32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        codes, scales = ops.quantize_rows(x.float())
        ops.int8_matmul(codes, scales, w, sw, out=out)
    for i in range(3):
        x.copy_(product(m, n, k, seed=i)[0])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.int8_matmul(*ops.quantize_rows(x.float()), w, sw, dtype=F32))


# ---------------------------------------------------------------- together

def test_a_prompt_and_the_tokens_after_it():
    """A recurrent layer as a program runs it: the prompts' activations to codes, one int8 projection for q, k, v and
    the gates, the rule over the prompts, then token by token; against float64 from the projection's codes on."""
    d, hk, hv, dk, dv = 256, 2, 4, 64, 64
    width = 2 * hk * dk + hv * dv
    lens, steps = [150, 3, 64], 4
    r = gen(3)
    w, sw = ops.quantize_rows(torch.randn(width + 2 * hv, d, generator=r, device="cuda") / d ** 0.5)
    x = torch.randn(sum(lens) + 3 * steps, d, generator=r, device="cuda").to(BF16)

    def project(rows):
        codes, sx = ops.quantize_rows(rows)
        y = ops.int8_matmul(codes, sx, w[:width], sw[:width], dtype=BF16)
        gates = ops.int8_matmul(codes, sx, w[width:], sw[width:], dtype=F32)
        n = rows.shape[0]
        check(y, *ops_f64.matmul(codes, sx, w[:width], sw[:width], None, BF16), "projection")
        return (y[:, :hk * dk].view(n, hk, dk), y[:, hk * dk:2 * hk * dk].view(n, hk, dk), y[:, 2 * hk * dk:].view(n, hv, dv),
                -torch.nn.functional.softplus(gates[:, :hv]), torch.sigmoid(gates[:, hv:]))

    S = torch.zeros(3, hv, dk, dv, device="cuda")
    cu = torch.tensor([0, 150, 153, 217], dtype=torch.int32, device="cuda")
    prompt = project(x[:217])
    outs = [ops.delta_chunk(*prompt, cu, state_in=S, state_out=S, normalize=True)]
    rows = [prompt]
    for t in range(steps):
        rows.append(project(x[217 + 3 * t:220 + 3 * t]))
        outs.append(ops.delta_step(*rows[-1], S, normalize=True))
    for i, (a, b) in enumerate([(0, 150), (150, 153), (153, 217)]):
        seq = [torch.cat([p[a:b]] + [s[i:i + 1] for s in parts]) for p, *parts in zip(*rows)]
        want, S64, tol, S_tol = ops_f64.rule(*seq, torch.zeros(hv, dk, dv, device="cuda"), normalize=True)
        check(torch.cat([outs[0][a:b]] + [o[i:i + 1] for o in outs[1:]]), want, tol, i)
        check(S[i], S64, S_tol, i)


# ---------------------------------------------------------------- the ends of f32's range

F32_MAX = torch.finfo(torch.float32).max


def one_column(x, cu, before, bad, col, head, normalize, changed, pool=None):
    """Of a call whose inputs `changed` from x in one column of a head, from row `bad` of the first sequence on: everything else
    has the bits of the call on x, and that column the rule's values.

    Beside ops_f64's bound stands one for factors that leave f32's range at its other end.  Over the tokens of a chunk a value V is
    multiplied by decays e^(G_i - G_j), of which what is below 2^-126 is 0: each of the entries of A, at most 1 in size, is off by 2^-126,
    so T = (I + A)^-1 by |T| |dA| |T| <= 64 * 64 * 2^-126 with |T| <= 1; limbs below 2^-126 add three such steps.  The result is then
    off by V * 2^-114 at most (|q|, |k| and the scale are at most 1), which is seen only where V is next to f32's end.
    """
    floor = 2.0 ** -114 * max(float(changed[2][:, head, col].abs().max()), 0.0 if pool is None else float(pool[0, head, :, col].abs().max()))
    S, S2 = torch.empty_like(before), torch.empty_like(before)
    want = ops.delta_chunk(*x, cu, state_in=before, state_out=S, normalize=normalize)
    start = before if pool is None else pool
    got = ops.delta_chunk(*changed, cu, state_in=start, state_out=S2, normalize=normalize)
    end = int(cu[1])
    exact, S64, tol, S_tol = ops_f64.rule(*(t[:end] for t in changed), start[0], normalize=normalize)
    check(got[bad:end, head, col], exact[bad:, head, col], tol[bad:, head, col] + floor, "out")
    check(S2[0, head, :, col], S64[head, :, col], S_tol[head, :, col] + floor, "state")
    got[bad:end, head, col] = want[bad:end, head, col]
    S2[0, head, :, col] = S[0, head, :, col]
    assert torch.equal(got, want) and torch.equal(S2, S)


ENDS = [(64, [130, 70]), (128, [130, 70]), (64, [50]), (128, [64]), (64, [101] + [5] * 70)]
ends = pytest.mark.parametrize("dk,lens", ENDS, ids=["64", "128", "64 rows at most", "64 rows at most, 128", "71 sequences"])


@ends
@pytest.mark.parametrize("size", [F32_MAX, -F32_MAX, 3.3962e38])
@pytest.mark.parametrize("at", [0, 29, 48])
def test_delta_chunk_of_a_value_next_to_the_end_of_f32(at, size, dk, lens):
    """It is finite, and so is what the rule makes of it."""
    x = rule_inputs(sum(lens), 2, 4, dk, 64, F32, seed=2, normalize=True)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    y = [t.clone() for t in x]
    y[2][at, 1, 5] = size
    one_column(x, cu, pool_of(len(lens), 4, dk, 64), at, 5, 1, True, y)


@ends
@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
@pytest.mark.parametrize("size", [F32_MAX, -F32_MAX])
def test_delta_chunk_of_a_state_next_to_the_end_of_f32(size, dtype, dk, lens):
    x = rule_inputs(sum(lens), 2, 4, dk, 64, dtype, seed=2)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    before = pool_of(len(lens), 4, dk, 64)
    pool = before.clone()
    pool[0, 1, 3, 5] = size
    one_column(x, cu, before, 0, 5, 1, False, x, pool)


@ends
def test_delta_chunk_of_a_query_next_to_the_end_of_f32(dk, lens):
    x = rule_inputs(sum(lens), 2, 4, dk, 64, F32, seed=2)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    before = 1e-3 * pool_of(len(lens), 4, dk, 64)
    x[2] *= 1e-3
    y = [t.clone() for t in x]
    at = 33
    y[0][at, 0, 7] = F32_MAX
    want, got = (ops.delta_chunk(*t, cu, state_in=before) for t in (x, y))
    exact, _, tol, _ = ops_f64.rule(*(t[:lens[0]] for t in y), before[0])
    check(got[at, :2], exact[at, :2], tol[at, :2], "out")
    got[at, :2] = want[at, :2]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
@pytest.mark.parametrize("which", ["k", "q"])
@pytest.mark.parametrize("lens,at", [([50], 20), ([130, 70], 64)])
def test_sums_of_squares_past_f32_are_not_finite_in_either_form(lens, at, which, dtype):
    """A key or query of finite values that cannot be normalized in f32, in a sequence and token by token."""
    hk, hv, dk, dv, T = 2, 4, 64, 64, sum(lens)
    x = rule_inputs(T, hk, hv, dk, dv, dtype, seed=2, normalize=True)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    before = pool_of(len(lens), hv, dk, dv)
    S, S2 = torch.empty_like(before), torch.empty_like(before)
    want = ops.delta_chunk(*x, cu, state_in=before, state_out=S, normalize=True)
    y = [t.clone() for t in x]
    y[which == "k"][at, 1] = 1e19
    got = ops.delta_chunk(*y, cu, state_in=before, state_out=S2, normalize=True)
    bad = torch.zeros(T, hv, dtype=torch.bool, device="cuda")
    bad[at:lens[0] if which == "k" else at + 1, 2:] = True
    assert not torch.isfinite(got[bad]).any() and torch.equal(got[~bad], want[~bad])
    if which == "k":
        assert not torch.isfinite(S2[0, 2:]).any()
        S2[0, 2:] = S[0, 2:]
    assert torch.equal(S2, S)
    # the same token by itself
    a, b = (before[:1].clone() for _ in range(2))
    want, got = (ops.delta_step(*(t[at:at + 1] for t in z), s, normalize=True) for z, s in ((x, a), (y, b)))
    assert not torch.isfinite(got[:, 2:]).any() and torch.equal(got[:, :2], want[:, :2])
    if which == "k":
        assert not torch.isfinite(b[0, 2:]).any()
        b[0, 2:] = a[0, 2:]
    assert torch.equal(a, b)


def test_the_largest_key_that_normalizes():
    """|k|^2 next to f32's end: still the rule's values."""
    x = rule_inputs(100, 1, 2, 64, 64, F32, seed=4, normalize=True)
    for t in (x[0], x[1]):
        t *= 1.8e19 / t.norm(dim=-1, keepdim=True)
    before = pool_of(1, 2, 64, 64)
    S, step = torch.empty_like(before), before.clone()
    out = ops.delta_chunk(*x, torch.tensor([0, 100], dtype=torch.int32, device="cuda"), state_in=before, state_out=S, normalize=True)
    want, S64, tol, S_tol = ops_f64.rule(*x, before[0], normalize=True)
    check(out, want, tol, "out")
    check(S[0], S64, S_tol, "state")
    for t in range(100):
        check(ops.delta_step(*(z[t:t + 1] for z in x), step, normalize=True), want[t:t + 1], tol[t:t + 1], t)
    check(step[0], S64, S_tol, "state by steps")


def test_quantize_rows_whose_scale_rounds_to_zero():
    """Largest values on both sides of 127 * 2^-150, half of f32's smallest step: below it the rounded scale is 0, as a row of zeros'
    is, and 1 stands in its place."""
    step = 2.0 ** -149
    most = [0, 1, 2, 17, 63, 64, 127, 200]
    x = torch.zeros(len(most), 70, device="cuda")
    for r, m in enumerate(most):
        x[r, 0], x[r, 3], x[r, 69] = m * step, -m * step, (m // 2) * step
    codes, scales = ops.quantize_rows(x)
    for r, m in enumerate(most):
        if m < 64:
            assert scales[r] == 1.0 and not codes[r].any(), m
        else:
            assert scales[r] == round(m / 127) * step and codes[r, 0] == 127 and codes[r, 3] == -127, m
