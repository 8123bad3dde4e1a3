"""e4m3 codes with a scale a block, and their product (quantize_blocks, fp8_matmul), on the GPU, against 64-bit
statements of them (tests/more_ops_f64.py)."""
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


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def refused(call):
    with pytest.raises(ffi.BackendError) as e:
        call()
    assert e.value.result == ffi.BackendResult.INVALID_ARGUMENT


def activations(rows, cols, dtype, seed=0):
    x = torch.randn(rows, cols, generator=gen(seed), device="cuda") * torch.exp(torch.randn(rows, 1, generator=gen(seed + 1), device="cuda"))
    x[:, ::37] *= 20.0
    return x.to(dtype)


def same_codes(x, block_rows, codes, scales):
    want, s = f64.quantize_blocks(x.float().cpu().numpy(), block_rows)
    assert np.array_equal(scales.cpu().numpy(), s)
    got = codes.float().cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.nan_to_num(got), np.nan_to_num(want))


@types
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 127), (5, 129), (127, 16), (128, 128), (129, 256), (300, 200), (2, 4096), (260, 1000)])
def test_quantize_blocks(rows, cols, block_rows, dtype):
    x = activations(rows, cols, dtype, seed=rows + cols)
    same_codes(x, block_rows, *ops.quantize_blocks(x, block_rows=block_rows))


@types
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("off,pad", [(1, 0), (0, 3), (8, 8), (4, 12)])
def test_quantize_blocks_strided_and_unaligned(off, pad, block_rows, dtype):
    rows, cols = 140, 264
    wide = activations(rows, cols + off + pad, dtype)
    x = wide[:, off:off + cols]
    held = torch.zeros(rows, cols + off + pad, dtype=torch.uint8, device="cuda")
    codes, scales = ops.quantize_blocks(x, block_rows=block_rows, codes=held.view(torch.float8_e4m3fn)[:, off:off + cols])
    same_codes(x, block_rows, codes, scales)
    assert (held[:, :off] == 0).all() and (held[:, off + cols:] == 0).all()


@types
def test_quantize_blocks_of_what_is_not_finite_and_of_zeros(dtype):
    x = activations(130, 256, dtype)
    x[0, 5], x[1, 200], x[2, 3], x[2, 9], x[3], x[4, :128] = NAN, INF, -INF, NAN, 0.0, NAN
    for block_rows in (1, 128):
        codes, scales = ops.quantize_blocks(x, block_rows=block_rows)
        same_codes(x, block_rows, codes, scales)
    codes, scales = ops.quantize_blocks(x)
    assert scales[1, 1] == INF and codes[1, 200 - 0].float().isnan() and (codes[1, 128:200].float() == 0).all()
    assert scales[3, 0] == 2.0 ** -126 and (codes[3].float() == 0).all()


def test_quantize_blocks_of_the_smallest_and_largest():
    """Blocks whose scale would be below 2^-126 take that; f32's largest value becomes 448."""
    tiny = torch.tensor([1e-45, 1e-40, 2.0 ** -126, 448 * 2.0 ** -126, 3e-36, 3.4028234e38], device="cuda")
    x = torch.zeros(6, 128, device="cuda")
    x[:, 0], x[:, 1] = tiny, -tiny / 3
    codes, scales = ops.quantize_blocks(x)
    same_codes(x, 1, codes, scales)
    assert codes[5, 0].float() == 448 and (scales[:4, 0] == 2.0 ** -126).all()


def test_quantize_blocks_rounds_halves_to_even():
    """Every border of two codes, with a scale of 1."""
    v = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    mid = (v[:-1] + v[1:]) / 2
    x = torch.cat([v, mid, torch.nextafter(mid, torch.tensor(1e9)), torch.nextafter(mid, torch.tensor(-1e9))])
    x = torch.cat([x, -x, torch.zeros(-2 * len(x) % 127)]).view(-1, 127)
    x = torch.cat([x, torch.full((len(x), 1), 448.0)], 1).cuda()
    codes, scales = ops.quantize_blocks(x)
    assert (scales == 1).all()
    same_codes(x, 1, codes, scales)


def test_quantize_blocks_more_units_than_one_dimension_of_a_launch():
    """More than 2^20 workgroups."""
    rows = 16 * (1 << 20) + 37
    x = torch.zeros(rows, 8, dtype=BF16, device="cuda")
    x[-1, 3], x[rows // 2, 0] = 4.0, 448.0
    codes, scales = ops.quantize_blocks(x)
    assert codes[-1, 3].float() == 448 and codes[rows // 2, 0].float() == 448 and scales[rows // 2, 0] == 1
    assert int((codes.view(torch.uint8) != 0).sum()) == 2


# ---------------------------------------------------------------- product

def product(m, n, k, seed=0):
    g = gen(seed)
    kb, nb = -(-k // 128), -(-n // 128)

    def codes(rows):
        return (torch.randn(rows, k, generator=g, device="cuda") * 100.0).clamp(-448, 448).to(torch.float8_e4m3fn)

    return [codes(m), torch.exp(torch.randn(m, kb, generator=g, device="cuda")) / 100.0, codes(n),
            torch.exp(torch.randn(nb, kb, generator=g, device="cuda")) / (100.0 * max(k, 1) ** 0.5)]


def check(got, x, bias, dtype, what=None):
    y, tol = f64.fp8_matmul(*x, bias, dtype)
    off = (got.double() - y).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((off / tol.clamp(min=1e-300)).max()))


SHAPES = [(1, 1, 16), (1, 16, 128), (1, 300, 768), (2, 129, 144), (3, 8200, 128), (4, 8200, 256), (5, 64, 272), (15, 128, 4096), (16, 200, 1040),
          (17, 200, 640), (33, 256, 128), (63, 64, 384), (64, 129, 256), (65, 65, 65 * 16), (100, 4096, 1536), (128, 768, 4096), (129, 1000, 768),
          (1000, 1536, 768), (1030, 2050, 400), (1100, 4100, 128), (2048, 4096, 256), (4100, 4200, 144), (4096, 4352, 128)]


@types
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_fp8_matmul(m, n, k, dtype):
    x = product(m, n, k, seed=m + n)
    bias = torch.randn(n, generator=gen(5), device="cuda") if (m + n) % 2 else None
    check(ops.fp8_matmul(*x, bias=bias, dtype=dtype), x, bias, dtype)


@types
@pytest.mark.parametrize("m,n,k,off,pad", [(1, 300, 17, 0, 0), (70, 200, 1, 0, 0), (70, 130, 200, 0, 3), (5, 130, 128, 16, 1), (130, 257, 130, 1, 1),
                                           (100, 96, 256, 16, 16), (20, 96, 272, 32, 0)])
def test_fp8_matmul_strided_and_unaligned(m, n, k, off, pad, dtype):
    x = product(m, n, k)
    wide = [torch.zeros(r, off + k + pad, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for r in (m, n)]
    for w, c in zip(wide, (x[0], x[2])):
        w.view(torch.uint8).fill_(0x7f)         # (NaN around the operands)
        w[:, off:off + k] = c
    out = torch.full((m, n + 5), 7.0, dtype=dtype, device="cuda")
    got = ops.fp8_matmul(wide[0][:, off:off + k], x[1], wide[1][:, off:off + k], x[3], out=out[:, 1:n + 1])
    check(got, x, None, dtype)
    assert (out[:, 0] == 7.0).all() and (out[:, n + 1:] == 7.0).all()


@types
def test_fp8_matmul_without_columns(dtype):
    x = product(3, 5, 0)
    assert (ops.fp8_matmul(*x, dtype=dtype) == 0).all()
    bias = torch.arange(5.0, device="cuda")
    assert torch.equal(ops.fp8_matmul(*x, bias=bias, dtype=dtype), bias.to(dtype).expand(3, 5))
    assert ops.fp8_matmul(*product(0, 5, 128)).shape == (0, 5) and ops.fp8_matmul(*product(5, 0, 128)).shape == (5, 0)


@types
@pytest.mark.parametrize("m,n", [(1, 200), (20, 200), (300, 520), (2100, 4100)])
def test_fp8_matmul_nan_stays_in_its_row_and_channel(m, n, dtype):
    x = product(m, n, 272)
    want = ops.fp8_matmul(*x, dtype=dtype)
    x[0][m // 2, 271] = NAN
    x[2][n // 3, 16] = NAN
    got = ops.fp8_matmul(*x, dtype=dtype)
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    bad[m // 2] = True
    bad[:, n // 3] = True
    assert got[bad].isnan().all() and torch.equal(got[~bad], want[~bad])


def test_fp8_matmul_16_bit_outputs_are_within_what_the_instruction_cuts_off():
    """One product that is larger than all others by 2^13 and more: the seven beside it may go, and no others."""
    m, n, k = 32, 64, 128
    x = product(m, n, k)
    x[0].fill_(1.0)
    x[2].fill_(1.0)
    x[0][:, 40], x[2][:, 40] = 256.0, 256.0
    x[1].fill_(1.0)
    x[3].fill_(1.0)
    exact = 65536.0 + 127
    assert (ops.fp8_matmul(*x, dtype=F32) == exact).all()
    x[1].fill_(2.0 ** -12)
    got = ops.fp8_matmul(*x, dtype=F16).float()
    assert ((got - exact * 2.0 ** -12).abs() <= 2.0 ** -12 * 7 + 2.0 ** -11 * 16).all()


@pytest.mark.parametrize("m,n,k", [(1, 300, 768), (20, 400, 768), (600, 1200, 256), (2100, 4100, 144)])
def test_fp8_matmul_captured(m, n, k):
    x = product(m, n, k)
    out = torch.empty(m, n, dtype=BF16, device="cuda")
    g = torch.cuda.CUDAGraph()
    ops.fp8_matmul(*x, out=out)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        ops.fp8_matmul(*x, out=out)
    for i in range(3):
        x[0].copy_(product(m, n, k, seed=i + 1)[0])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.fp8_matmul(*x))


@pytest.mark.parametrize("of", ["x", "w", "out"])
def test_fp8_matmul_offsets_past_32_bits(of):
    """Operands and outputs of more than 2^32 bytes: the last rows are as right as the first."""
    m, n, k = {"x": (9 * 2 ** 17, 64, 4096), "w": (17, 9 * 2 ** 17, 4096), "out": (70000, 32768, 128)}[of]
    x = product(256, 256, k)
    reps = lambda t, rows: t.repeat(-(-rows // t.shape[0]), 1)[:rows]  # noqa: E731
    y = [reps(x[0], m), reps(x[1], m), reps(x[2], n), reps(x[3], -(-n // 128))]
    got = ops.fp8_matmul(*y)
    for i, j in ((0, 0), (m - 17, n - 64)):
        part = got[i:i + 17, j:j + 64]
        full = [y[0][i:i + 17], y[1][i:i + 17], y[2][j:j + 64], y[3][j // 128:j // 128 + 1]]
        assert (j + 63) // 128 == j // 128
        check(part, full, None, BF16, (i, j))


def test_a_layer_in_8_bits_from_prompt_to_token():
    """quantize_blocks -> fp8_matmul -> scan_chunk -> quantize_blocks -> fp8_matmul -> sample, then a token with scan_step: as a program
    runs them, against the same steps in 64 bits from the codes on."""
    T, d, ch, n, vocab = 90, 256, 192, 16, 1000
    g = gen(3)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    w_in, w_out = randn(2 * ch + 32 + ch, d) / d ** 0.5, randn(vocab, ch) / ch ** 0.5
    wi, wis = ops.quantize_blocks(w_in, block_rows=128)
    wo, wos = ops.quantize_blocks(w_out, block_rows=128)
    a, dd, bias = -torch.exp(randn(ch, n) * 0.3), 1 + 0.1 * randn(ch), randn(ch) - 3.0
    pool = torch.zeros(1, ch, n, device="cuda")
    u = torch.tensor([0.37], device="cuda")

    def forward(x, scan):
        q, s = ops.quantize_blocks(x)
        p = ops.fp8_matmul(q, s, wi, wis, dtype=F32)
        xs, z, bc, dt = p[:, :ch], p[:, ch:2 * ch], p[:, 2 * ch:2 * ch + 32], p[:, 2 * ch + 32:]
        y = scan(x=xs, z=z, dt=dt, a=a, b=bc[:, :n].unflatten(1, (1, n)), c=bc[:, n:].unflatten(1, (1, n)), d=dd, dt_bias=bias)
        q2, s2 = ops.quantize_blocks(y)
        logits = ops.fp8_matmul(q2[-1:], s2[-1:], wo, wos, dtype=F32)
        return p, y, (q2, s2), logits, ops.sample(logits, u, temperature=0.8, top_k=50, top_p=0.9)

    x = randn(T, d)
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    p, y, (q2, s2), logits, token = forward(x, lambda **k: ops.scan_chunk(cu_seqlens=cu, state_in=pool, state_out=pool, **k))
    q, s = ops.quantize_blocks(x)
    want, tol = f64.fp8_matmul(q, s, wi, wis, None, F32)
    assert ((p.double() - want).abs() <= tol).all()
    out, h = f64.scan(x=p[:, :ch], z=p[:, ch:2 * ch], dt=p[:, 2 * ch + 32:], a=a, b=p[:, 2 * ch:2 * ch + n].unflatten(1, (1, n)),
                      c=p[:, 2 * ch + n:2 * ch + 32].unflatten(1, (1, n)), d=dd, dt_bias=bias, h0=torch.zeros(ch, n, device="cuda"))
    v, tol = f64.rounded(out, F32)
    assert ((y.double() - v).abs() <= tol).all()
    want, tol = f64.fp8_matmul(q2[-1:], s2[-1:], wo, wos, None, F32)
    assert ((logits.double() - want).abs() <= tol).all()
    assert int(token) == f64.draw(logits[0].cpu().numpy(), 0.37, 0.8, 50, 0.9)
    p1, y1, _, _, token1 = forward(randn(1, d), lambda **k: ops.scan_step(states=pool, **k))
    out, h = f64.scan(x=p1[:, :ch], z=p1[:, ch:2 * ch], dt=p1[:, 2 * ch + 32:], a=a, b=p1[:, 2 * ch:2 * ch + n].unflatten(1, (1, n)),
                      c=p1[:, 2 * ch + n:2 * ch + 32].unflatten(1, (1, n)), d=dd, dt_bias=bias, h0=h.v)
    v, tol = f64.rounded(out, F32)
    assert torch.allclose(y1.double(), v, rtol=1e-4, atol=1e-5) and 0 <= int(token1) < vocab
