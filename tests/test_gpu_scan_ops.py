"""The selective scan on caller tensors (scan_step, scan_chunk, scan_grad, scan) on the GPU, against 64-bit
statements of it (tests/more_ops_f64.py)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from redukt_amd import ffi, ops  # noqa: E402
from tests import more_ops_f64 as f64  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
NAMES = {BF16: "bf16", F16: "f16", F32: "f32"}
types = pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=NAMES.get)
sizes = pytest.mark.parametrize("n", [8, 16, 32, 64])
GRADS = ("x", "dt", "a", "b", "c", "d", "z", "dt_bias", "state_in")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def layer(T, ch, n, groups, dtype, seed=0, step=1.0):
    """Inputs by name; step: what the time steps are multiplied by."""
    r = gen(seed)
    randn = lambda *s: torch.randn(*s, generator=r, device="cuda")  # noqa: E731
    s = step * torch.exp(torch.rand(ch, generator=r, device="cuda") * 4.6 - 5.0)
    return {"x": randn(T, ch).to(dtype), "dt": (0.7 * randn(T, ch)).to(dtype),
            "a": -torch.arange(1, n + 1, device="cuda") * torch.exp(0.1 * randn(ch, n)), "b": randn(T, groups, n).to(dtype),
            "c": randn(T, groups, n).to(dtype), "d": 1.0 + 0.1 * randn(ch), "z": randn(T, ch).to(dtype),
            "dt_bias": s + torch.log(-torch.expm1(-s))}


def pool_of(slots, ch, n, seed=5):
    return 0.5 * torch.randn(slots, ch, n, generator=gen(seed), device="cuda")


def rows_of(x, r):
    return {k: v[r] if k in ("x", "dt", "b", "c", "z") and v is not None else v for k, v in x.items()}


def cu_of(lens, start=0):
    return torch.tensor(start + np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def check(got, want, dtype, what):
    v, tol = f64.rounded(want, dtype)
    off = (got.double() - v).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((off / tol.clamp(min=1e-300)).max()), float(off.max()))


def refused(call):
    with pytest.raises(ffi.BackendError) as e:
        call()
    assert e.value.result == ffi.BackendResult.INVALID_ARGUMENT


# ---------------------------------------------------------------- one token

@types
@sizes
@pytest.mark.parametrize("rows,ch,groups", [(1, 1, 1), (1, 192, 1), (3, 70, 1), (17, 128, 2), (40, 16, 1)])
def test_scan_step(rows, ch, groups, n, dtype):
    x = layer(rows, ch, n, groups, dtype, seed=rows + n)
    pool = pool_of(rows + 2, ch, n)
    slots = torch.from_numpy(np.random.default_rng(rows).permutation(rows + 2)[:rows].astype(np.int32)).cuda()
    before = pool.clone()
    out = ops.scan_step(states=pool, slots=slots, **x)
    for s in set(range(rows + 2)) - set(slots.tolist()):
        assert torch.equal(pool[s], before[s])
    for i, s in enumerate(slots.tolist()):
        want, h = f64.scan(h0=before[s], **rows_of(x, slice(i, i + 1)))
        check(out[i:i + 1], want, dtype, ("out", i))
        check(pool[s], h, F32, ("state", i))


@pytest.mark.parametrize("left", [("z",), ("d",), ("dt_bias",), ("z", "d", "dt_bias")], ids=str)
def test_scan_step_without(left):
    x = dict(layer(5, 40, 16, 1, F32), **{k: None for k in left})
    pool = pool_of(5, 40, 16)
    before = pool.clone()
    out = torch.empty(5, 40, device="cuda")
    assert ops.scan_step(states=pool, out=out, **x) is out
    for i in range(5):
        want, h = f64.scan(h0=before[i], **rows_of(x, slice(i, i + 1)))
        check(out[i:i + 1], want, F32, i)
        check(pool[i], h, F32, i)


@types
def test_scan_step_slices_of_projections(dtype):
    """x and z as halves of one projection's rows, B and C behind a time step's rank in another's, at odd places; out into a wider buffer."""
    rows, ch, n = 6, 33, 16
    x = layer(rows, ch, n, 1, dtype, seed=3)
    xz = torch.cat([x["x"], x["z"]], 1)
    dbc = torch.cat([torch.zeros(rows, 3, dtype=dtype, device="cuda"), x["b"].flatten(1), x["c"].flatten(1)], 1)
    wide = torch.full((rows, ch + 5), 7.0, dtype=dtype, device="cuda")
    p, q = pool_of(rows, ch, n), pool_of(rows, ch, n)
    y = dict(x, x=xz[:, :ch], z=xz[:, ch:], b=dbc[:, 3:3 + n].unflatten(1, (1, n)), c=dbc[:, 3 + n:].unflatten(1, (1, n)))
    got = ops.scan_step(states=p, out=wide[:, :ch], **y)
    assert torch.equal(got, ops.scan_step(states=q, **x)) and torch.equal(p, q) and (wide[:, ch:] == 7.0).all()


def test_scan_step_padded_bad_and_repeated_slots():
    rows, ch, n = 7, 20, 16
    x = layer(rows, ch, n, 1, F32)
    for k in ("x", "dt", "z", "b", "c"):
        x[k][1] = float("nan")              # a padded entry may hold anything
    pool = pool_of(4, ch, n)
    before = pool.clone()
    out = torch.full((rows, ch), 7.0, device="cuda")
    slots = torch.tensor([2, -1, 4, 0, 2, -7, -1], dtype=torch.int32, device="cuda")
    ops.scan_step(states=pool, slots=slots, out=out, **x)
    for i in (0, 3):
        want, h = f64.scan(h0=before[int(slots[i])], **rows_of(x, slice(i, i + 1)))
        check(out[i:i + 1], want, F32, i)
        check(pool[int(slots[i])], h, F32, i)
    assert (out[[1, 6]] == 7.0).all() and out[[2, 4, 5]].isnan().all() and torch.equal(pool[[1, 3]], before[[1, 3]])


def test_scan_step_offsets_past_32_bits():
    """A pool of more than 2^31 values: the last slot is stepped as the first one is."""
    ch, n = 1536, 64
    slots = 2 ** 31 // (ch * n) + 2
    pool = torch.empty(slots, ch, n, device="cuda")
    pool[0] = pool_of(1, ch, n)[0]
    pool[-1] = pool[0]
    x = {k: v.repeat(2, *[1] * (v.dim() - 1)) if k in ("x", "dt", "z", "b", "c") else v for k, v in layer(1, ch, n, 1, BF16).items()}
    out = ops.scan_step(states=pool, slots=torch.tensor([0, slots - 1], dtype=torch.int32, device="cuda"), **x)
    assert torch.equal(out[0], out[1]) and torch.equal(pool[0], pool[-1])
    want, h = f64.scan(h0=pool_of(1, ch, n)[0], **rows_of(x, slice(0, 1)))
    check(out[:1], want, BF16, "out")
    check(pool[-1], h, F32, "state")


# ---------------------------------------------------------------- sequences

def sequences(lens, ch, n, groups, dtype, initial, before_rows=0, behind=0, seed=0, step=1.0, left=()):
    T = sum(lens)
    x = dict(layer(before_rows + T + behind, ch, n, groups, dtype, seed=seed, step=step), **{k: None for k in left})
    k = len(lens)
    slots = torch.from_numpy(np.random.default_rng(seed).permutation(k + 2)[:k].astype(np.int32)).cuda()
    first = pool_of(k + 2, ch, n) if initial else None
    last = torch.full((k + 2, ch, n), 7.0, device="cuda")
    out = torch.full((before_rows + T + behind, ch), 7.0, dtype=dtype, device="cuda")
    ops.scan_chunk(cu_seqlens=cu_of(lens, before_rows), state_in=first, state_out=last, slots=slots, out=out, **x)
    at = before_rows
    for i, (length, s) in enumerate(zip(lens, slots.tolist())):
        want, h = f64.scan(h0=first[s] if initial else torch.zeros(ch, n, device="cuda"), **rows_of(x, slice(at, at + length)))
        check(out[at:at + length], want, dtype, ("out", i))
        check(last[s], h, F32, ("state", i))
        at += length
    assert (out[:before_rows] == 7.0).all() and (out[before_rows + T:] == 7.0).all()
    for s in set(range(k + 2)) - set(slots.tolist()):
        assert (last[s] == 7.0).all()


@types
@pytest.mark.parametrize("lens", [[1], [3], [4], [15], [16], [17], [32], [33], [63], [64], [65], [128], [130], [200], [1, 64, 0, 3, 129, 0]],
                         ids=lambda v: "-".join(map(str, v)))
@pytest.mark.parametrize("ch,n", [(40, 16), (17, 64)])
def test_scan_chunk_lengths(lens, ch, n, dtype):
    sequences(lens, ch, n, 1, dtype, initial=True, before_rows=2, behind=3, seed=len(lens) + lens[0])


@types
@sizes
@pytest.mark.parametrize("ch,groups", [(1, 1), (192, 3), (100, 1)])
def test_scan_chunk_sizes(ch, groups, n, dtype):
    sequences([70, 1, 130], ch, n, groups, dtype, initial=False, seed=n)


@pytest.mark.parametrize("left", [("z",), ("d",), ("dt_bias",), ("z", "d", "dt_bias")], ids=str)
def test_scan_chunk_without(left):
    sequences([70, 20], 40, 16, 1, F32, initial=True, left=left)


@pytest.mark.parametrize("step", [1e-3, 30.0])
@pytest.mark.parametrize("lens", [[2300], [1900]], ids=str)
def test_scan_chunk_long(lens, step):
    """Long memories and short ones; one by a launch that joins the pieces, one whose pieces join themselves."""
    sequences(lens, 24, 16, 1, F32, initial=True, step=step)


def test_scan_chunk_alone_and_among_others():
    """A sequence's bits depend on nothing else in the call, whichever way its pieces are joined."""
    ch, n, lens = 70, 16, [300, 5, 900, 64, 1500]
    x = layer(sum(lens), ch, n, 1, BF16)
    first, last = pool_of(5, ch, n), torch.empty(5, ch, n, device="cuda")
    out = ops.scan_chunk(cu_seqlens=cu_of(lens), state_in=first, state_out=last, **x)
    at = 0
    for i, length in enumerate(lens):
        one = torch.empty(1, ch, n, device="cuda")
        r = slice(at, at + length)
        alone = ops.scan_chunk(cu_seqlens=cu_of([length]), state_in=first[i:i + 1], state_out=one, **rows_of(x, r))
        assert torch.equal(out[r], alone) and torch.equal(last[i], one[0]), i
        at += length


@types
@sizes
def test_scan_chunk_of_single_tokens_is_scan_step(n, dtype):
    x = layer(9, 48, n, 1, dtype)
    p, q = pool_of(9, 48, n), pool_of(9, 48, n)
    a = ops.scan_step(states=p, **x)
    b = ops.scan_chunk(cu_seqlens=cu_of([1] * 9), state_in=q, state_out=q, **x)
    assert torch.equal(a, b) and torch.equal(p, q)


@pytest.mark.parametrize("lens", [[50, 3], [700, 64], [2500, 0, 3]], ids=str)
def test_scan_chunk_in_place(lens):
    """The pool's first states are read before its last ones are written."""
    x = layer(sum(lens), 40, 16, 1, F32)
    p = pool_of(len(lens), 40, 16)
    want = torch.empty_like(p)
    a = ops.scan_chunk(cu_seqlens=cu_of(lens), state_in=p.clone(), state_out=want, **x)
    b = ops.scan_chunk(cu_seqlens=cu_of(lens), state_in=p, state_out=p, **x)
    assert torch.equal(a, b) and torch.equal(p, want)


@pytest.mark.parametrize("long", [70, 2200])
def test_scan_chunk_padded_bad_and_repeated_slots(long):
    lens = [long, 5, 6, long, 7, 8]
    ch, n = 20, 16
    x = layer(sum(lens), ch, n, 1, F32)
    pool = pool_of(3, ch, n)
    before = pool.clone()
    out = torch.full((sum(lens), ch), 7.0, device="cuda")
    slots = torch.tensor([1, -1, 3, 1, 2, -5], dtype=torch.int32, device="cuda")
    ops.scan_chunk(cu_seqlens=cu_of(lens), state_in=pool, state_out=pool, slots=slots, out=out, **x)
    at = np.concatenate([[0], np.cumsum(lens)])
    for i in range(6):
        r = slice(at[i], at[i + 1])
        if i in (0, 4):
            want, h = f64.scan(h0=before[int(slots[i])], **rows_of(x, r))
            check(out[r], want, F32, i)
            check(pool[int(slots[i])], h, F32, i)
        elif i == 1:
            assert (out[r] == 7.0).all()
        else:
            assert out[r].isnan().all()
    assert torch.equal(pool[0], before[0])
    # without states to write, sequences may share a slot
    same = torch.ones(6, dtype=torch.int32, device="cuda")
    out = ops.scan_chunk(cu_seqlens=cu_of(lens), state_in=before, slots=same, **x)
    want, _ = f64.scan(h0=before[1], **rows_of(x, slice(at[4], at[5])))
    check(out[at[4]:at[5]], want, F32, "shared")


@pytest.mark.parametrize("long", [100, 2200])
def test_scan_chunk_what_is_not_finite(long):
    """One of x in its channel from its token on, one of B in its group's channels, one of C or z in its token."""
    ch, n, groups = 128, 16, 2
    x = layer(long, ch, n, groups, F32)
    cu = cu_of([10, long - 10])
    want = ops.scan_chunk(cu_seqlens=cu, **x)
    for name, at, hit in (("x", (40, 3), (slice(40, None), slice(3, 4))), ("dt", (40, 3), (slice(40, None), slice(3, 4))),
                          ("b", (40, 1, 2), (slice(40, None), slice(64, None))), ("c", (40, 1, 2), (slice(40, 41), slice(64, None))),
                          ("z", (40, 5), (slice(40, 41), slice(5, 6)))):
        for bad in (float("nan"), float("inf")):
            y = dict(x, **{name: x[name].clone()})
            y[name][at] = bad
            if name == "z" and bad > 0:
                continue                     # (an open gate's output is the infinity times the sum)
            got = ops.scan_chunk(cu_seqlens=cu, **y)
            mask = torch.zeros(long, ch, dtype=torch.bool, device="cuda")
            mask[hit] = True
            assert torch.equal(got[~mask], want[~mask]), (name, bad)
            if bad != bad or name != "dt":
                assert not torch.isfinite(got[mask]).any(), (name, bad)


def test_scan_chunk_time_steps_of_minus_infinity():
    """Such a token leaves the state as it is."""
    x = layer(150, 20, 16, 1, F32)
    x["dt"][[5, 64, 65, 149]] = float("-inf")
    keep = [t for t in range(150) if t not in (5, 64, 65, 149)]
    first = pool_of(1, 20, 16)
    a, b = torch.empty_like(first), torch.empty_like(first)
    out = ops.scan_chunk(cu_seqlens=cu_of([150]), state_in=first, state_out=a, **x)
    y = {k: v[keep].contiguous() if k in ("x", "dt", "z", "b", "c") else v for k, v in x.items()}
    ops.scan_chunk(cu_seqlens=cu_of([146]), state_in=first, state_out=b, **y)
    assert torch.allclose(a, b, rtol=1e-4, atol=1e-5) and torch.isfinite(out).all()
    before = f64.scan(h0=first[0], **rows_of(x, slice(0, 150)))[1]
    check(a[0], before, F32, "state")


def test_scan_chunk_odd_boundaries():
    """Boundaries that decrease or leave the rows touch nothing outside the arrays; sequences in order before them are right."""
    x = layer(200, 20, 16, 1, F32)
    want = ops.scan_chunk(cu_seqlens=cu_of([70, 30]), **rows_of(x, slice(0, 100)))
    guard = torch.full((202, 20), 7.0, device="cuda")
    for tail in ([100, 50], [100, 90, 1000], [100, -5, 3], [100, 2 ** 31 - 1]):
        cu = torch.tensor([0, 70] + tail, dtype=torch.int32, device="cuda")
        states = torch.zeros(len(cu) - 1, 20, 16, device="cuda")
        ops.scan_chunk(cu_seqlens=cu, out=guard[1:201], state_out=states, **x)
        assert torch.equal(guard[1:71], want[:70]) and (guard[0] == 7.0).all() and (guard[201] == 7.0).all()


def test_scan_chunk_captured_and_on_another_stream():
    lens = [300, 2, 2100]
    x = layer(sum(lens), 70, 16, 1, BF16)
    cu = cu_of(lens)
    a, b = pool_of(3, 70, 16), pool_of(3, 70, 16)
    out = torch.empty(sum(lens), 70, dtype=BF16, device="cuda")
    work = torch.empty(ops.scan_chunk_workspace(sum(lens), 3, 70, 1, 16), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    ops.scan_chunk(cu_seqlens=cu, state_in=a, state_out=a, out=out, workspace=work, stream=side.cuda_stream, **x)
    side.synchronize()
    first = ops.scan_chunk(cu_seqlens=cu, state_in=b, state_out=b, **x)
    assert torch.equal(out, first) and torch.equal(a, b)
    refused(lambda: ops.scan_chunk(cu_seqlens=cu, stream=side.cuda_stream, **x))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.scan_chunk(cu_seqlens=cu, state_in=a, state_out=a, out=out, workspace=work, **x)
    for i in range(4):
        if i == 2:                           # other lengths of the same buffers
            cu.copy_(cu_of([64, 0, 1900]))
        g.replay()
        torch.cuda.synchronize()
        want = ops.scan_chunk(cu_seqlens=cu, state_in=b, state_out=b, **x)
        rows = int(cu[-1])
        assert torch.equal(out[:rows], want[:rows]) and torch.equal(a, b)


# ---------------------------------------------------------------- gradients

def gradients(lens, ch, n, groups, dtype, initial=True, final=True, before_rows=0, behind=0, seed=0, step=1.0, left=()):
    T = before_rows + sum(lens) + behind
    x = dict(layer(T, ch, n, groups, dtype, seed=seed, step=step), **{k: None for k in left})
    dout = torch.randn(T, ch, generator=gen(seed + 9), device="cuda").to(dtype)
    first = pool_of(len(lens), ch, n) if initial else None
    dlast = pool_of(len(lens), ch, n, seed=8) if final else None
    got = ops.scan_grad(dout, cu_seqlens=cu_of(lens, before_rows), state_in=first, dstate_out=dlast, **x)
    zero = torch.zeros(ch, n, device="cuda")
    at, sums = before_rows, None
    for i, length in enumerate(lens):
        r = slice(at, at + length)
        want = f64.scan_grad(dout[r], h0=first[i] if initial else zero, dfinal=dlast[i] if final else zero, **rows_of(x, r))
        for k in ("x", "dt", "z", "b", "c"):
            if x[k] is not None:
                check(getattr(got, k)[r], want[k], dtype, (k, i))
        if initial:
            check(got.state_in[i], want["state_in"], F32, ("state_in", i))
        part = {k: want[k] for k in ("a", "d", "dt_bias")}
        sums = part if sums is None else {k: sums[k] + part[k] for k in part}
        at += length
    for k in ("a", "d", "dt_bias"):
        if x[k] is not None:
            check(getattr(got, k), sums[k], F32, k)
    for k in GRADS:
        if k == "state_in":
            assert (got.state_in is None) == (not initial)
        else:
            assert (getattr(got, k) is None) == (x[k] is None)
    for k in ("x", "dt", "z", "b", "c"):
        if x[k] is not None:
            assert (getattr(got, k)[:before_rows] == 0).all() and (getattr(got, k)[at:] == 0).all()


@types
@pytest.mark.parametrize("lens", [[1], [3], [4], [16], [17], [32], [63], [64], [65], [130], [200], [1, 64, 0, 3, 129, 0]],
                         ids=lambda v: "-".join(map(str, v)))
@pytest.mark.parametrize("ch,n", [(40, 16), (17, 64)])
def test_scan_grad_lengths(lens, ch, n, dtype):
    gradients(lens, ch, n, 1, dtype, before_rows=2, behind=70, seed=len(lens) + lens[0])


@types
@sizes
@pytest.mark.parametrize("ch,groups", [(1, 1), (192, 3), (300, 1)])
def test_scan_grad_sizes(ch, groups, n, dtype):
    gradients([70, 1, 130], ch, n, groups, dtype, initial=False, final=False, seed=n)


@pytest.mark.parametrize("left", [("z",), ("d",), ("dt_bias",), ("z", "d", "dt_bias")], ids=str)
@pytest.mark.parametrize("initial,final", [(True, False), (False, True)])
def test_scan_grad_without(left, initial, final):
    gradients([70, 20], 40, 16, 1, F32, initial=initial, final=final, left=left)


@pytest.mark.parametrize("step", [1e-3, 30.0])
@pytest.mark.parametrize("lens", [[2300], [1900]], ids=str)
def test_scan_grad_long(lens, step):
    gradients(lens, 24, 16, 1, F32, step=step)


def test_scan_grad_many_channels():
    """Several blocks of channels a workgroup (enough pieces of them), whose sums meet."""
    gradients([300] * 12, 640, 16, 1, F32, seed=3)


def test_scan_grad_without_rows():
    x = layer(0, 20, 16, 1, F32)
    dlast = pool_of(2, 20, 16)
    got = ops.scan_grad(torch.empty(0, 20, device="cuda"), cu_seqlens=cu_of([0, 0]), state_in=pool_of(2, 20, 16, seed=1), dstate_out=dlast, **x)
    assert torch.equal(got.state_in, dlast) and (got.a == 0).all() and (got.d == 0).all() and (got.dt_bias == 0).all()
    y = layer(5, 20, 16, 1, F32)
    got = ops.scan_grad(torch.ones(5, 20, device="cuda"), cu_seqlens=cu_of([]), **y)
    assert all((g == 0).all() for g in got if g is not None)


@pytest.mark.parametrize("lens", [[90, 40], [2200, 7]], ids=str)
def test_scan_grad_against_differences(lens):
    """Along random directions of every input: the 64-bit scan's central difference."""
    ch, n = 24, 16
    x = layer(sum(lens), ch, n, 1, F32, seed=4)
    first, dlast = pool_of(2, ch, n), pool_of(2, ch, n, seed=8)
    dout = torch.randn(sum(lens), ch, generator=gen(9), device="cuda")
    got = ops.scan_grad(dout, cu_seqlens=cu_of(lens), state_in=first, dstate_out=dlast, **x)

    def loss(y, h0):
        total, at = 0.0, 0
        for i, length in enumerate(lens):
            out, h = f64.scan(h0=h0[i], **rows_of(y, slice(at, at + length)))
            total += float((out.v * dout[at:at + length].double()).sum() + (h.v * dlast[i].double()).sum())
            at += length
        return total

    wide = {k: v.double() for k, v in x.items()}
    for k in GRADS:
        base = first.double() if k == "state_in" else wide[k]
        v = torch.randn(base.shape, generator=gen(11), device="cuda", dtype=torch.float64)
        eps = 1e-5
        args = [(dict(wide), base + sg * eps * v) if k == "state_in" else (dict(wide, **{k: base + sg * eps * v}), first.double()) for sg in (1, -1)]
        want = (loss(*args[0]) - loss(*args[1])) / (2 * eps)
        g = getattr(got, k).double()
        # the difference's own error is about eps^2 of the third derivative; f32's that of the gradients' bound, 1e-5 of the magnitudes summed
        assert abs(float((g * v).sum()) - want) <= 1e-5 * float((g * v).abs().sum()) + 1e-6 * abs(want), k


def test_scan_grad_is_the_same_every_time_and_captured():
    lens = [300, 2, 2100]
    T, ch, n = sum(lens), 130, 16
    x = layer(T, ch, n, 1, BF16)
    cu, dout = cu_of(lens), torch.randn(T, ch, device="cuda").to(BF16)
    first = pool_of(3, ch, n)
    want = ops.scan_grad(dout, cu_seqlens=cu, state_in=first, **x)
    grads = ops.ScanGrads(*(torch.empty_like(g) for g in want))
    work = torch.empty(ops.scan_grad_workspace(T, 3, ch, 1, n), dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.scan_grad(dout, cu_seqlens=cu, state_in=first, grads=grads, workspace=work, **x)
    for i in range(4):
        dout.normal_()
        g.replay()
        torch.cuda.synchronize()
        want = ops.scan_grad(dout, cu_seqlens=cu, state_in=first, **x)
        assert all(torch.equal(p, q) for p, q in zip(want, grads)), i


def test_scan_grad_strided():
    """Slices of projections in and out."""
    T, ch, n = 75, 33, 16
    x = layer(T, ch, n, 1, BF16)
    dout = torch.randn(T, ch, device="cuda").to(BF16)
    want = ops.scan_grad(dout, cu_seqlens=cu_of([75]), **x)
    xz = torch.cat([x["x"], x["z"]], 1)
    dxz, dbc = torch.full((T, 2 * ch + 1), 7.0, dtype=BF16, device="cuda"), torch.full((T, 2 * n + 3), 7.0, dtype=BF16, device="cuda")
    grads = ops.ScanGrads(x=dxz[:, :ch], z=dxz[:, ch:2 * ch], b=dbc[:, 3:3 + n].unflatten(1, (1, n)), c=dbc[:, 3 + n:].unflatten(1, (1, n)),
                          dt=torch.empty_like(want.dt), a=torch.empty_like(want.a), d=torch.empty_like(want.d),
                          dt_bias=torch.empty_like(want.dt_bias), state_in=None)
    got = ops.scan_grad(dout, cu_seqlens=cu_of([75]), grads=grads, **dict(x, x=xz[:, :ch], z=xz[:, ch:]))
    assert all(p is None and q is None or torch.equal(p, q) for p, q in zip(want, got))
    assert (dxz[:, 2 * ch:] == 7.0).all() and (dbc[:, :3] == 7.0).all()


# ---------------------------------------------------------------- autograd

def test_scan_is_scan_chunk_and_scan_grad():
    lens = [70, 30]
    x = layer(100, 40, 16, 1, F32)
    first = pool_of(2, 40, 16)
    leaves = {k: v.clone().requires_grad_() for k, v in x.items()}
    h0 = first.clone().requires_grad_()
    out, last = ops.scan(cu_seqlens=cu_of(lens), state_in=h0, **leaves)
    last_want = torch.empty_like(first)
    assert torch.equal(out, ops.scan_chunk(cu_seqlens=cu_of(lens), state_in=first, state_out=last_want, **x)) and torch.equal(last, last_want)
    dout, dlast = torch.randn_like(out), torch.randn_like(last)
    ((out * dout).sum() + (last * dlast).sum()).backward()
    want = ops.scan_grad(dout, cu_seqlens=cu_of(lens), state_in=first, dstate_out=dlast, **x)
    for k in GRADS:
        assert torch.equal((h0 if k == "state_in" else leaves[k]).grad, getattr(want, k)), k
    # an output alone, and a part of the inputs
    y = dict(x, b=x["b"].clone().requires_grad_(), d=None, z=None, dt_bias=None)
    out, last = ops.scan(cu_seqlens=cu_of(lens), **y)
    (g,) = torch.autograd.grad(last.sum(), [y["b"]])
    want = ops.scan_grad(torch.zeros_like(out), cu_seqlens=cu_of(lens), dstate_out=torch.ones_like(last), **dict(y, b=x["b"]))
    assert torch.equal(g, want.b)


def test_scan_of_a_projection_and_an_expanded_gradient():
    """Inputs that are views of one projection, a gradient of stride 0, B used by two layers: gradients add up."""
    T, ch, n = 60, 32, 16
    x = layer(T, ch, n, 1, F32)
    xz = torch.cat([x["x"], x["z"]], 1).requires_grad_()
    b = x["b"].clone().requires_grad_()
    for _ in range(2):
        out, _ = ops.scan(cu_seqlens=cu_of([T]), **dict(x, x=xz[:, :ch], z=xz[:, ch:], b=b))
        out.sum().backward()
    want = ops.scan_grad(torch.ones(T, ch, device="cuda"), cu_seqlens=cu_of([T]), **x)
    assert torch.equal(xz.grad, 2 * torch.cat([want.x, want.z], 1)) and torch.equal(b.grad, 2 * want.b)


def test_scan_notices_what_was_overwritten():
    x = {k: v.requires_grad_() for k, v in layer(20, 32, 16, 1, F32).items()}
    out, _ = ops.scan(cu_seqlens=cu_of([20]), **x)
    with torch.no_grad():
        x["x"].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_scan_of_a_padded_batch():
    """Rows of no sequence: zeros, with gradients of zero, whatever was in the memory and is in their inputs."""
    lens, before, behind, ch = [70, 0, 9], 3, 40, 48
    T = before + sum(lens) + behind
    x = layer(T, ch, 16, 1, F32)
    live = slice(before, before + sum(lens))
    for k in ("x", "dt", "z", "b", "c"):
        x[k][:before] = x[k][live.stop:] = float("nan")
    filler = torch.full((T, ch), float("nan"), device="cuda")
    del filler                               # (its memory is likely the output's)
    leaves = {k: v.clone().requires_grad_() for k, v in x.items()}
    out, _ = ops.scan(cu_seqlens=cu_of(lens, before), **leaves)
    assert (out[:before] == 0).all() and (out[live.stop:] == 0).all()
    assert torch.equal(out[live], ops.scan_chunk(cu_seqlens=cu_of(lens), **rows_of(x, live)))
    mask = torch.zeros(T, 1, device="cuda")
    mask[live] = 1.0
    (out * mask).square().sum().backward()
    for k, v in leaves.items():
        assert v.grad.isfinite().all(), k
        if k in ("x", "dt", "z", "b", "c"):
            assert (v.grad[:before] == 0).all() and (v.grad[live.stop:] == 0).all(), k


def test_scan_captured_with_its_backward_pass():
    """Leaves that no eager pass has seen; every replay against the operators themselves."""
    lens = [150, 1, 40]
    T, ch = sum(lens), 64
    x = layer(T, ch, 16, 1, F32)
    cu, dout = cu_of(lens), torch.randn(T, ch, device="cuda")
    names = [k for k in GRADS if k != "state_in"]
    leaves = {k: x[k].clone().requires_grad_() for k in names}
    ops.scan_grad(dout, cu_seqlens=cu, **x)  # (kernels are loaded by their first call)
    ops.scan_chunk(cu_seqlens=cu, **x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, last = ops.scan(cu_seqlens=cu, **leaves)
        grads = torch.autograd.grad([out], [leaves[k] for k in names], [dout])
    for i in range(4):
        with torch.no_grad():
            leaves["x"].normal_(), leaves["b"].normal_(), dout.normal_()
        g.replay()
        torch.cuda.synchronize()
        now = {k: v.detach() for k, v in leaves.items()}
        final = torch.empty_like(last)
        assert torch.equal(out.detach(), ops.scan_chunk(cu_seqlens=cu, state_out=final, **now)) and torch.equal(last.detach(), final), i
        want = ops.scan_grad(dout, cu_seqlens=cu, **now)
        assert all(torch.equal(p, getattr(want, k)) for k, p in zip(names, grads)), i


def test_scan_on_two_streams_at_once():
    lens = [2100, 300]
    T, ch, n = sum(lens), 200, 16
    both = []
    for seed in (1, 2):
        x = layer(T, ch, n, 1, BF16, seed=seed)
        dout = torch.randn(T, ch, generator=gen(seed + 20), device="cuda").to(BF16)
        want = ops.scan_grad(dout, cu_seqlens=cu_of(lens), **x)
        both.append((x, dout, cu_of(lens), ops.scan_chunk(cu_seqlens=cu_of(lens), **x), want, torch.zeros(T, ch, dtype=BF16, device="cuda"),
                     ops.ScanGrads(*(None if g is None else torch.zeros_like(g) for g in want)),
                     torch.empty(ops.scan_chunk_workspace(T, 2, ch, 1, n), dtype=torch.uint8, device="cuda"),
                     torch.empty(ops.scan_grad_workspace(T, 2, ch, 1, n), dtype=torch.uint8, device="cuda"), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for x, dout, cu, _, _, out, grads, work, back, on in both:
            ops.scan_chunk(cu_seqlens=cu, out=out, workspace=work, stream=on.cuda_stream, **x)
            ops.scan_grad(dout, cu_seqlens=cu, grads=grads, workspace=back, stream=on.cuda_stream, **x)
    torch.cuda.synchronize()
    for _, _, _, first, want, out, grads, *_ in both:
        assert torch.equal(out, first) and all(p is None and q is None or torch.equal(p, q) for p, q in zip(want, grads))


def test_a_prompt_and_the_tokens_after_it():
    """scan_chunk, then scan_step from the states that it left."""
    ch, n, T = 96, 16, 200
    x = layer(T, ch, n, 1, F32, seed=6)
    pool = torch.zeros(3, ch, n, device="cuda")
    slot = torch.tensor([2], dtype=torch.int32, device="cuda")
    rows = [ops.scan_chunk(cu_seqlens=cu_of([190]), state_in=pool, state_out=pool, slots=slot, **rows_of(x, slice(0, 190)))]
    rows += [ops.scan_step(states=pool, slots=slot, **rows_of(x, slice(t, t + 1))) for t in range(190, T)]
    want, h = f64.scan(h0=torch.zeros(ch, n, device="cuda"), **x)
    check(torch.cat(rows), want, F32, "out")
    check(pool[2], h, F32, "state")
    assert (pool[:2] == 0).all()
