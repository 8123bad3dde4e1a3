"""Every way that the sizes of a call choose through the scan and its gradients, fp8_matmul and sample, on the GPU, against the 64-bit
statements of tests/more_ops_f64.py.  (That the shapes here choose those ways: test_op_ways_host.py.)"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from redukt_amd import ops  # noqa: E402
from tests import more_ops_f64 as f64  # noqa: E402
from tests.test_gpu_fp8_ops import check, product  # noqa: E402
from tests.test_gpu_sample import SETTINGS, logits_of, uniform  # noqa: E402
from tests.test_gpu_scan_ops import check as scan_check, gradients, layer, pool_of, rows_of, sequences  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF16, F16, F32]
NAMES = {BF16: "bf16", F16: "f16", F32: "f32"}
types = pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
INF, NAN = float("inf"), float("nan")

# ---------------------------------------------------------------- the scan

STEPS = [(45, 1100, 1), (70, 768, 2), (800, 17, 1)]        # entries, channels, groups: enough of them for 64 channels a wave


@types
@pytest.mark.parametrize("n", [8, 16, 32, 64])
@pytest.mark.parametrize("rows,ch,groups", STEPS)
def test_scan_step_of_many_channels(rows, ch, groups, n, dtype):
    """Channels past the last whole 64, padded entries, slots out of range and named twice, states that no entry names."""
    x = layer(rows, ch, n, groups, dtype, seed=rows + n)
    slots = np.random.default_rng(rows).permutation(rows + 2)[:rows].astype(np.int32)
    slots[5], slots[7], slots[8], slots[11] = -1, rows + 2, -9, slots[3]
    pool = pool_of(rows + 2, ch, n)
    before = pool.clone()
    out = torch.full((rows, ch), 7.0, dtype=dtype, device="cuda")
    ops.scan_step(states=pool, slots=torch.from_numpy(slots).cuda(), out=out, **x)
    assert (out[5] == 7.0).all() and out[[7, 8, 11]].isnan().all()
    named = sorted(set(range(rows)) - {5, 7, 8, 11})
    free = sorted(set(range(rows + 2)) - {int(slots[i]) for i in named})
    assert torch.equal(pool[free], before[free])
    for i in named[::max(1, rows // 40)] + [named[-1]]:
        want, h = f64.scan(h0=before[int(slots[i])], **rows_of(x, slice(i, i + 1)))
        scan_check(out[i:i + 1], want, dtype, ("out", i))
        scan_check(pool[int(slots[i])], h, F32, ("state", i))


CHUNKS = [([2200, 0, 70, 3], True), ([900, 64, 1, 33], False)]      # lengths; whether a launch of its own joins the pieces


@types
@pytest.mark.parametrize("n", [8, 16, 32, 64])
@pytest.mark.parametrize("lens,joined", CHUNKS, ids=["joined", "by-themselves"])
def test_scan_chunk_of_many_pieces(lens, joined, n, dtype):
    sequences(lens, 70, n, 1, dtype, initial=True, before_rows=2, behind=3, seed=n)


# Many sequences, most of them of one piece: places in the workspace go by rows.  (The second half: those of more follow each other closely.)
SPREAD = [([1] * 300 + [130, 64, 65, 0, 200, 33] + [2] * 40, False), ([1] * 200 + [2200, 3, 65, 66] + [0] * 30, True),
          ([65, 65, 66, 129, 65] * 3 + [1] * 40, False), ([33, 33, 34, 65, 33] * 4 + [0, 1] * 30, False)]


@types
@pytest.mark.parametrize("n", [16, 64])
@pytest.mark.parametrize("way", range(len(SPREAD)))
def test_scan_chunk_of_many_sequences(way, n, dtype):
    sequences(SPREAD[way][0], 70, n, 1, dtype, initial=True, before_rows=way, behind=3, seed=n)


@pytest.mark.parametrize("way", range(len(SPREAD)))
def test_scan_chunk_of_many_sequences_in_place_and_alone(way):
    """The same bits in place, and of each long sequence in a call of its own (whose places go by sequences)."""
    lens = SPREAD[way][0]
    x = layer(sum(lens), 70, 16, 1, BF16)
    cu = torch.from_numpy(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)).cuda()
    first, last = pool_of(len(lens), 70, 16), torch.empty(len(lens), 70, 16, device="cuda")
    want = ops.scan_chunk(cu_seqlens=cu, state_in=first, state_out=last, **x)
    pool = first.clone()
    assert torch.equal(ops.scan_chunk(cu_seqlens=cu, state_in=pool, state_out=pool, **x), want) and torch.equal(pool, last)
    for i, n in enumerate(lens):
        if n > 64:
            r, one = slice(int(cu[i]), int(cu[i + 1])), torch.empty(1, 70, 16, device="cuda")
            alone = ops.scan_chunk(cu_seqlens=torch.tensor([0, n], dtype=torch.int32, device="cuda"), state_in=first[i:i + 1], state_out=one, **rows_of(x, r))
            assert torch.equal(alone, want[r]) and torch.equal(one[0], last[i]), i


# ---------------------------------------------------------------- gradients of the scan

# lengths, channels, groups; then by states of up to 16 parts and of more: blocks of channels that a workgroup takes, whether a launch
# of its own joins the pieces.  None is small enough for the shorter pieces, but the last two.
GRAD_WAYS = {
    "four-blocks": ([5] * 200 + [150, 0, 64, 65, 200], 1100, 1, ((4, False), (4, True))),
    "four-blocks-few-rows": ([2] * 250 + [100, 64, 33, 250], 1100, 1, ((4, False), (4, False))),
    "four-blocks-of-two-groups": ([4] * 250 + [130, 70], 768, 2, ((4, False), (4, True))),
    "two-or-four-blocks-joined": ([1] * 450 + [1100, 130, 700, 129], 500, 1, ((2, True), (4, True))),
    "a-block-each-joined": ([70] * 40, 640, 1, ((1, True), (1, True))),
    "a-block-each": ([100] * 10, 1100, 1, ((1, False), (1, False))),
    "many-in-short-pieces": ([1] * 30 + [33, 65, 0, 40, 66] + [2] * 9, 70, 1, ((1, False), (1, False))),
    "many-in-short-pieces-joined": ([1] * 50 + [1100, 33], 70, 1, ((1, True), (1, True))),
}
SHORT_WAYS = {"many-in-short-pieces", "many-in-short-pieces-joined"}


def grad_way(lens, ch, groups, n):
    """(short pieces, blocks of a workgroup, joined by a launch, bytes of workspace) as scan_grad's plan has them."""
    rows, blocks, piece = sum(lens), -(-(ch // groups) // 64), 64 if n <= 16 else 32
    short = (rows // piece + len(lens)) * blocks * groups < 384
    piece //= 2 if short else 1
    pieces, per = rows // piece + len(lens) + 2, 4
    while per > 1 and pieces * groups * -(-blocks // per) < 1024:
        per //= 2
    places = min(pieces, 2 * rows // piece)     # (for sequences of more than one piece)
    floats = places * ch * (2 * n + 1) + pieces * ch * (n + 2) + -(-blocks // per) * groups * rows * 2 * n + 12
    return short, per, rows > 32 * piece, 4 * floats


@types
@pytest.mark.parametrize("n", [8, 16, 32, 64])
def test_scan_grad_of_four_blocks_a_workgroup(n, dtype):
    lens, ch, groups, _ = GRAD_WAYS["four-blocks"]
    gradients(lens, ch, n, groups, dtype, before_rows=3, behind=70, seed=n)


@pytest.mark.parametrize("i,n", enumerate([8, 16, 32, 64]))
@pytest.mark.parametrize("j,way", enumerate(w for w in GRAD_WAYS if w != "four-blocks"))
def test_scan_grad_ways(way, n, i, j):
    lens, ch, groups, _ = GRAD_WAYS[way]
    gradients(lens, ch, n, groups, TYPES[(i + j) % 3], seed=n + j)


# ---------------------------------------------------------------- products

# More blocks of 128 columns than any tile has stages, and a part of one at the end.
DEEP = [(16, 200, 1040), (2, 20000, 656), (100, 400, 1168), (600, 1200, 1168), (600, 1700, 1168), (1000, 2100, 1168), (2048, 4096, 1040),
        (4100, 4200, 656), (130, 257, 650)]


@types
@pytest.mark.parametrize("m,n,k", DEEP)
def test_fp8_matmul_of_many_blocks(m, n, k, dtype):
    x = product(m, n, k, seed=m + n)
    bias = torch.randn(n, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    check(ops.fp8_matmul(*x, bias=bias, dtype=dtype), x, bias, dtype)


def any_codes(rows, k, seed):
    """Codes of every finite value alike: products next to each other differ by up to 2^35, subnormal ones among them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = torch.randint(0, 254, (rows, k), generator=g, device="cuda", dtype=torch.int16)
    return (c + (c >= 127).to(torch.int16)).to(torch.uint8).view(torch.float8_e4m3fn)      # (0x7f and 0xff are NaN)


@types
@pytest.mark.parametrize("m,n,k", [(5, 300, 768), (40, 300, 768), (300, 520, 784), (600, 1200, 400), (33, 70, 401)])
def test_fp8_matmul_of_codes_of_all_sizes(m, n, k, dtype):
    x = product(m, n, k)
    x[0], x[2] = any_codes(m, k, 1), any_codes(n, k, 2)
    check(ops.fp8_matmul(*x, dtype=dtype), x, None, dtype)


@types
@pytest.mark.parametrize("m", [3, 70, 2100])
def test_fp8_matmul_of_large_codes_that_cancel(m, dtype):
    """448 x 448 twice, with both signs, and small products whose sum is 6: in the same eight columns as those, where 16-bit outputs may be off
    by what seven products are cut off by; then each of the three in an eight of its own, where nothing is."""
    n, k = 200 if m < 2000 else 4200, 144
    one = torch.ones(m, 2, device="cuda"), torch.ones(-(-n // 128), 2, device="cuda")
    for apart in (1, 8):
        for first in (0, 96, 120, 128 - 16):
            x, w = torch.zeros(m, k, device="cuda"), torch.zeros(n, k, device="cuda")
            x[:, first], x[:, first + apart] = 448.0, -448.0
            w[:, first], w[:, first + apart] = 448.0, 448.0
            at = slice(first + 2, first + 8) if apart == 1 else slice(first + 16, first + 22)
            x[:, at] = w[:, at] = 1.0
            args = x.to(torch.float8_e4m3fn), one[0], w.to(torch.float8_e4m3fn), one[1]
            got = ops.fp8_matmul(*args, dtype=dtype)
            if dtype == F32 or apart == 8:
                assert (got == 6.0).all(), (apart, first)
            else:
                check(got, args, None, dtype, first)
                assert (got <= 6.0).all()


# ---------------------------------------------------------------- sampling

def drawn(logits, u, **settings):
    rows = logits.float().cpu().numpy()
    return [f64.draw_fast(rows[i], float(u[i]), **{k: v[i].item() if isinstance(v, torch.Tensor) else v for k, v in settings.items()})
            for i in range(len(rows))]


@types
@pytest.mark.parametrize("vocab", [50280, 70001, 131072])
def test_sample_of_large_vocabularies_few_rows_and_many(vocab, dtype):
    """Masked, tied and nearly equal logits and NaN, in rows that begin at any place, for workgroups of either size."""
    rows, times = 8, 40
    wide = logits_of(rows, vocab + 3, dtype, seed=vocab)
    x = wide[:, 1:vocab + 1]
    x[1] = -INF
    x[2, ::2] = -INF
    x[3] = 1.5
    x[4] = torch.linspace(1.0, 1.01, vocab, device="cuda").to(dtype)
    x[5, ::3] = NAN
    x[6] = torch.arange(vocab, device="cuda").remainder(7).to(dtype)
    y = x.contiguous()
    for i, s in enumerate(SETTINGS):
        u = uniform(rows, seed=i)
        want = drawn(x, u, **s)
        for t in (x, y):
            assert ops.sample(t, u, **s).tolist() == want, s
            assert ops.sample(t.repeat(times, 1), u.repeat(times), **s).tolist() == want * times, s
