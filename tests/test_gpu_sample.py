"""Tokens drawn from logits (sample) on the GPU: the same ones as a row-by-row statement in 64 bits and whole
numbers (tests/more_ops_f64.py) draws."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from redukt_amd import ffi, ops  # noqa: E402
from tests import more_ops_f64 as f64  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
NAMES = {BF16: "bf16", F16: "f16", F32: "f32"}
types = pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=NAMES.get)
INF, NAN = float("inf"), float("nan")


def logits_of(rows, vocab, dtype, seed=0, spread=2.5):
    r = np.random.default_rng(seed)
    x = r.standard_normal((rows, vocab)) * spread
    x[np.arange(rows), r.integers(0, vocab, rows)] += 4.0
    return torch.from_numpy(x.astype(np.float32)).cuda().to(dtype)


def drawn(logits, u, **settings):
    """What the statement draws; settings are numbers or tensors [rows]."""
    rows = logits.float().cpu().numpy()
    def at(v, i):
        return v[i].item() if isinstance(v, torch.Tensor) else v
    return [f64.draw(rows[i], u[i].item(), **{k: at(v, i) for k, v in settings.items() if v is not None}) for i in range(len(rows))]


def same(logits, u, **settings):
    got = ops.sample(logits, u, **settings)
    assert got.dtype == torch.int32 and got.tolist() == drawn(logits, u, **settings)
    return got


def uniform(rows, seed=1):
    return torch.from_numpy(np.random.default_rng(seed).random(rows, dtype=np.float32)).cuda()


SETTINGS = [{}, dict(temperature=0.7), dict(top_k=1), dict(top_k=5, temperature=1.5), dict(top_p=0.8), dict(min_p=0.05), dict(top_p=0.999),
            dict(top_k=40, top_p=0.9, min_p=0.02, temperature=0.9), dict(top_k=3000, top_p=0.95), dict(min_p=0.9), dict(temperature=0.0),
            dict(top_k=10 ** 9), dict(top_p=1e-6), dict(min_p=2.0), dict(top_p=0.0), dict(top_k=-3, top_p=2.0, min_p=-1.0)]


@types
@pytest.mark.parametrize("vocab", [1, 2, 7, 256, 1000, 4096, 4097, 5000, 50280])
def test_sample(vocab, dtype):
    rows = 5
    logits = logits_of(rows, vocab, dtype, seed=vocab)
    for i, s in enumerate(SETTINGS):
        same(logits, uniform(rows, seed=i), **s)


@types
def test_sample_with_settings_of_each_row(dtype):
    rows, vocab = 64, 3001
    r = np.random.default_rng(4)
    t = lambda v, d: torch.from_numpy(v.astype(d)).cuda()  # noqa: E731
    settings = dict(temperature=t(r.uniform(0.0, 2.0, rows) * (r.random(rows) > 0.1), np.float32), top_k=t(r.integers(-1, 100, rows), np.int32),
                    top_p=t(r.uniform(0.1, 1.2, rows), np.float32), min_p=t(r.uniform(-0.1, 0.3, rows), np.float32))
    same(logits_of(rows, vocab, dtype), uniform(rows), **settings)


@types
@pytest.mark.parametrize("vocab", [700, 40000])
def test_sample_of_many_equal_logits(vocab, dtype):
    """Ties at every border go by index: all equal, two values, and a few values each held by thousands."""
    r = np.random.default_rng(2)
    x = np.zeros((4, vocab), np.float32)
    x[1, ::3] = 1.0
    x[2] = r.integers(0, 4, vocab)
    x[3] = r.integers(0, 2, vocab) * 1e-3 + 5.0
    logits = torch.from_numpy(x).cuda().to(dtype)
    for i, s in enumerate([{}, dict(top_k=300), dict(top_k=vocab - 5), dict(top_p=0.5), dict(top_p=0.9999), dict(top_k=vocab // 2, top_p=0.7),
                           dict(top_k=vocab // 3, top_p=0.9, min_p=0.5), dict(min_p=1.0), dict(temperature=100.0, top_p=0.3)]):
        same(logits, uniform(4, seed=i), **s)


def test_sample_nearly_equal_logits():
    """Tens of thousands of different values in one bin of the search."""
    vocab = 30000
    x = torch.linspace(1.0, 1.001, vocab)[torch.from_numpy(np.random.default_rng(3).permutation(vocab))].cuda()[None].repeat(2, 1)
    for i, s in enumerate([{}, dict(top_k=12345), dict(top_p=0.37), dict(top_k=20000, top_p=0.61), dict(temperature=50.0, top_k=7)]):
        same(x, uniform(2, seed=i), **s)


@types
def test_sample_masked(dtype):
    """-inf, the type's lowest value and NaN; rows with nothing left, or one; +inf takes everything."""
    vocab = 5003
    low = torch.finfo(dtype).min
    x = logits_of(8, vocab, dtype)
    x[0, 100:] = -INF
    x[1] = -INF
    x[2, :] = NAN
    x[3, :] = -INF
    x[3, 4321] = -3.0
    x[4, ::2] = low
    x[5, ::3] = NAN
    x[6] = low
    x[7, [5, 77, 4000]] = INF
    for s in [{}, dict(top_k=50), dict(top_p=0.9), dict(min_p=0.1), dict(top_k=20, top_p=0.5, min_p=0.01), dict(temperature=0.0)]:
        for seed in range(3):
            got = same(x, uniform(8, seed=seed), **s).tolist()
            assert got[1] == got[2] == -1 and got[3] == 4321 and got[7] in (5, 77, 4000)


def test_sample_temperatures():
    """Very small, very large and infinite ones, NaN and below 0."""
    x = logits_of(6, 2000, F32)
    t = torch.tensor([1e-38, 1e-3, 1e30, INF, NAN, -1.0], device="cuda")
    for s in ({}, dict(top_k=30), dict(top_p=0.4), dict(min_p=0.3)):
        same(x, uniform(6), temperature=t, **s)
    x[3, :100] = -INF                       # (an infinite temperature makes all others alike)
    assert ops.sample(x, torch.zeros(6, device="cuda"), temperature=t)[3] == 100


def test_sample_random_numbers_at_the_ends():
    x = logits_of(6, 3000, F32)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 5.0, -1.0, NAN], device="cuda")
    for s in ({}, dict(top_k=30), dict(top_p=0.4)):
        same(x, u, **s)
    x[:, 0] = -INF
    x[:, 1] = 9.0
    assert ops.sample(x, torch.zeros(6, device="cuda")).tolist() == [1] * 6        # (0 is the first that weighs something)


def test_sample_every_token_of_a_flat_row():
    """Each of 1,024 equal tokens has its share of [0, 1), to the last step."""
    x = torch.zeros(1, 1024, device="cuda")
    for i in (0, 1, 511, 1023):
        lo, hi = i / 1024, np.nextafter(np.float32((i + 1) / 1024), np.float32(0))
        for u in (lo, hi):
            assert ops.sample(x, torch.tensor([u], device="cuda")).item() == i


@types
@pytest.mark.parametrize("off,pad", [(0, 3), (1, 0), (8, 8)])
def test_sample_strided_and_unaligned(off, pad, dtype):
    rows, vocab = 4, 5000
    wide = logits_of(rows, off + vocab + pad, dtype)
    wide[:, :off] = 50.0
    if pad:
        wide[:, off + vocab:] = 50.0
    x = wide[:, off:off + vocab]
    for s in ({}, dict(top_k=20), dict(top_p=0.9)):
        same(x, uniform(rows), **s)
    same(logits_of(1, vocab, dtype).expand(rows, vocab), uniform(rows))


@pytest.mark.parametrize("dtype", [BF16, F32], ids=NAMES.get)
@pytest.mark.parametrize("vocab", [131072, 1 << 20])
def test_sample_large_vocabularies(vocab, dtype):
    x = logits_of(2, vocab, dtype, spread=0.3)
    for s in ({}, dict(top_k=100), dict(top_p=0.9), dict(top_k=vocab // 2, top_p=0.99)):
        same(x, uniform(2), **s)


@types
@pytest.mark.parametrize("vocab", [1, 7, 1000, 5003, 50280, 70001, 131072])
def test_sample_of_few_rows_and_of_many(vocab, dtype):
    """A row's token does not depend on how many there are: masked rows, ties and nearly equal values, strided as well."""
    rows, times = 8, 40
    wide = logits_of(rows, vocab + 8, dtype, seed=vocab)
    x = wide[:, :vocab]
    x[1] = -INF
    x[2, ::2] = -INF
    x[3] = 1.5
    x[4] = torch.linspace(1.0, 1.01, vocab, device="cuda").to(dtype)
    x[5, ::3] = NAN
    for i, s in enumerate(SETTINGS):
        u = uniform(rows, seed=i)
        few = ops.sample(x, u, **s)
        many = ops.sample(wide.repeat(times, 1)[:, :vocab] if i % 2 else x.repeat(times, 1), u.repeat(times), **s)
        assert torch.equal(many, few.repeat(times)), s
        assert few.tolist() == drawn(x, u, **s) or vocab > 5003, s


def test_sample_offsets_past_32_bits():
    rows, vocab = 70000, 1 << 15
    x = torch.full((rows, vocab), -INF, dtype=BF16, device="cuda")
    at = (torch.arange(rows, device="cuda") * 7919) % vocab
    x.scatter_(1, at[:, None], 1.0)
    got = ops.sample(x, uniform(rows), top_k=10)
    assert torch.equal(got.long(), at)


def test_sample_rows_do_not_meet():
    x = logits_of(300, 1000, F32)
    u = uniform(300)
    got = ops.sample(x, u, top_k=50, top_p=0.9)
    for i in (0, 7, 299):
        assert ops.sample(x[i:i + 1], u[i:i + 1], top_k=50, top_p=0.9).item() == got[i].item()


def test_sample_frequencies():
    """A million draws of eight tokens: within five standard deviations of their shares."""
    p = torch.softmax(torch.tensor([0.0, 1.0, 2.0, -1.0, 0.5, -INF, 1.5, 2.5], dtype=torch.float64), 0)
    n = 1 << 20
    x = torch.tensor([[0.0, 1.0, 2.0, -1.0, 0.5, -INF, 1.5, 2.5]], device="cuda").expand(n, 8)
    count = torch.bincount(ops.sample(x, torch.rand(n, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")).long(), minlength=8).cpu()
    assert ((count - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all() and count[5] == 0


def test_sample_captured_and_on_another_stream():
    x, u = logits_of(9, 6000, BF16), uniform(9)
    k = torch.full((9,), 40, dtype=torch.int32, device="cuda")
    out = torch.empty(9, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    ops.sample(x, u, top_k=k, out=out, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out, ops.sample(x, u, top_k=k))
    with pytest.raises(ffi.BackendError):
        ops.sample(x, u, stream=side.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.sample(x, u, top_k=k, top_p=0.9, out=out)
    for i in range(4):
        u.copy_(uniform(9, seed=i + 5))
        k.fill_(10 + i)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.sample(x, u, top_k=k, top_p=0.9))


@types
@pytest.mark.parametrize("vocab", [2, 3, 900, 5001, 50280])
def test_sample_infinite_temperature_of_masked_rows(vocab, dtype):
    """All tokens that are not masked weigh the same, with every filter; the row's end is no token."""
    x = logits_of(5, vocab, dtype, seed=vocab)
    x[:, 1::2] = -INF
    t = torch.full((5,), INF, device="cuda")
    for i, s in enumerate([{}, dict(top_k=1), dict(top_k=300), dict(top_k=vocab - 1), dict(top_p=0.6), dict(top_k=40, top_p=0.5, min_p=1.0)]):
        got = same(x, uniform(5, seed=i), temperature=t, **s)
        assert (got % 2 == 0).all()
