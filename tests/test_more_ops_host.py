"""The selective scan, the block-scaled fp8 product and sampling on caller tensors, without a GPU: the header and its
Python mirror, what is refused before anything is launched, and the 64-bit statements that the GPU tests go by."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from redukt_amd import ffi, ops  # noqa: E402
from tests import more_ops_f64 as f64  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD, OK = int(ffi.BackendResult.INVALID_ARGUMENT), int(ffi.BackendResult.OK)
P = 1 << 20        # an aligned address that no call may reach
F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib():
    return ops._load()


def test_the_structs_are_the_headers(tmp_path):
    structs = {"redukt_scan_rows": ops.ScanRows, "redukt_scan_grads": ops.ScanGradients, "redukt_quantize_blocks": ops.QuantizeBlocks,
               "redukt_fp8_matmul": ops.Fp8Matmul, "redukt_sample": ops.Sample}
    lines, want = ["#include <stdio.h>", "#include <stddef.h>", '#include "redukt_ops.h"', "int main(void) {"], []
    for name, cls in structs.items():
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        want.append(ctypes.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append('printf("%%zu\\n", offsetof(%s, %s));' % (name, f))
            want.append(getattr(cls, f).offset)
    src = tmp_path / "s.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    exe = str(tmp_path / "s")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    assert [int(v) for v in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()] == want


def scan_rows(**over):
    v = dict(dtype=0, rows=4, channels=128, groups=2, n=16, x=P, dt=P, z=P, b=P, c=P, out=P, x_stride=128, dt_stride=128, z_stride=128,
             b_stride=32, c_stride=32, out_stride=128, a=P, d=P, dt_bias=P)
    v.update(over)
    return ops.ScanRows(**v)


def scan_grads(**over):
    v = dict(dout=P, dx=P, ddt=P, dz=P, db=P, dc=P, dout_stride=128, dx_stride=128, ddt_stride=128, dz_stride=128, db_stride=32, dc_stride=32,
             da=P, dd=P, ddt_bias=P)
    v.update(over)
    return ops.ScanGradients(**v)


SIZES = [dict(dtype=3), dict(rows=1 << 31), dict(channels=0), dict(channels=(1 << 20) + 64, groups=1), dict(groups=0), dict(groups=3),
         dict(groups=4), dict(n=0), dict(n=4), dict(n=24), dict(n=128)]
ROWS = SIZES + [dict(x=None), dict(dt=None), dict(b=None), dict(c=None), dict(a=None), dict(x=P + 1), dict(dt=P + 1), dict(z=P + 1), dict(b=P + 1),
                dict(c=P + 1), dict(a=P + 2), dict(d=P + 2), dict(dt_bias=P + 1), dict(x_stride=127), dict(dt_stride=0), dict(z_stride=-128),
                dict(b_stride=31), dict(c_stride=16), dict(x_stride=(1 << 22) + 1)]
OUT = [dict(out=None), dict(out=P + 1), dict(out_stride=127), dict(out_stride=1 << 30)]


@pytest.mark.parametrize("over", ROWS + OUT, ids=str)
def test_scan_rows_refused(lib, over):
    a = ctypes.byref(scan_rows(**over))
    assert lib.redukt_op_scan_step(a, P, 8, P, None) == BAD
    assert lib.redukt_op_scan_chunk(a, P, 2, P, P, 8, P, P, 1 << 40, None) == BAD
    if over not in OUT:
        g = ctypes.byref(scan_grads())
        assert lib.redukt_op_scan_grad(a, g, P, 2, P, P, P, P, 1 << 40, None) == BAD


def test_scan_step_refused(lib):
    a = ctypes.byref(scan_rows())
    call = lib.redukt_op_scan_step
    assert call(None, P, 8, P, None) == BAD
    assert call(a, None, 8, P, None) == BAD
    assert call(a, P + 8, 8, P, None) == BAD              # states unaligned
    assert call(a, P, 8, P + 2, None) == BAD              # slots unaligned
    assert call(a, P, 3, None, None) == BAD               # four entries, three slots
    assert call(a, P, 1 << 31, P, None) == BAD
    assert call(ctypes.byref(scan_rows(rows=65537)), P, 1 << 20, P, None) == BAD
    assert call(ctypes.byref(scan_rows(rows=0, x=None)), None, 0, None, None) == OK
    assert call(a, P, 8, P, None) == BAD                  # sizes are right, but no device owns the address


def test_scan_chunk_refused(lib):
    rows = scan_rows(rows=400)
    a, big = ctypes.byref(rows), 1 << 40
    call = lib.redukt_op_scan_chunk
    assert call(None, P, 2, P, P, 8, P, P, big, None) == BAD
    assert call(a, None, 2, P, P, 8, P, P, big, None) == BAD
    assert call(a, P + 2, 2, P, P, 8, P, P, big, None) == BAD
    assert call(a, P, 65537, P, P, 1 << 20, P, P, big, None) == BAD
    assert call(a, P, 2, P + 4, P, 8, P, P, big, None) == BAD
    assert call(a, P, 2, P, P + 1024, 8, P, P, big, None) == BAD         # pools that overlap in part
    assert call(a, P, 9, P, P, 8, None, P, big, None) == BAD             # nine sequences, eight slots
    assert call(a, P, 2, None, None, 0, P, P, big, None) == BAD          # slots of no pool
    assert call(a, P, 0, None, None, 0, None, None, 0, None) == OK
    need = lib.redukt_op_scan_chunk_workspace(a, 2)
    assert need > 0
    assert call(a, P, 2, P, P, 8, P, None, big, None) == BAD
    assert call(a, P, 2, P, P, 8, P, P + 4, big, None) == BAD
    assert call(a, P, 2, P, P, 8, P, P, need - 1, None) == BAD
    assert call(a, P, 2, P, P, 8, P, P, big, None) == BAD                # no device owns the address


def test_scan_grad_refused(lib):
    a, big = ctypes.byref(scan_rows()), 1 << 40
    call = lib.redukt_op_scan_grad
    g = ctypes.byref(scan_grads())
    assert call(None, g, P, 2, P, P, P, P, big, None) == BAD
    assert call(a, None, P, 2, P, P, P, P, big, None) == BAD
    for over in (dict(dout=None), dict(dx=None), dict(ddt=None), dict(dz=None), dict(db=None), dict(dc=None), dict(da=None), dict(dd=None),
                 dict(ddt_bias=None), dict(dx=P + 1), dict(da=P + 4), dict(dd=P + 2), dict(ddt_bias=P + 2), dict(dout_stride=127), dict(dx_stride=0),
                 dict(db_stride=31), dict(dc_stride=(1 << 22) + 1)):
        assert call(a, ctypes.byref(scan_grads(**over)), P, 2, P, P, P, P, big, None) == BAD, over
    for over, missing in ((dict(z=None), dict(dz=P)), (dict(d=None), dict(dd=P)), (dict(dt_bias=None), dict(ddt_bias=P))):
        assert call(ctypes.byref(scan_rows(**over)), ctypes.byref(scan_grads(**missing)), P, 2, P, P, P, P, big, None) == BAD
    assert call(a, g, None, 2, P, P, P, P, big, None) == BAD
    assert call(a, g, P + 2, 2, P, P, P, P, big, None) == BAD
    for states in ((P + 4, P, P), (P, P + 4, P), (P, P, P + 4)):
        assert call(a, g, P, 2, *states, P, big, None) == BAD
    need = lib.redukt_op_scan_grad_workspace(a, 2)
    assert need > 0
    assert call(a, g, P, 2, P, P, P, None, big, None) == BAD
    assert call(a, g, P, 2, P, P, P, P, need - 1, None) == BAD
    assert call(a, g, P, 65537, P, P, P, P, big, None) == BAD
    assert call(a, g, P, 2, P, P, P, P, big, None) == BAD                # no device owns the address


def test_workspaces_of_sizes_that_are_not_taken(lib):
    for f in (lib.redukt_op_scan_chunk_workspace, lib.redukt_op_scan_grad_workspace):
        for over in SIZES:
            assert f(ctypes.byref(scan_rows(**over)), 2) == 0
        assert f(None, 2) == 0 and f(ctypes.byref(scan_rows(rows=400)), 65537) == 0
    for f in (ops.scan_chunk_workspace, ops.scan_grad_workspace):
        sizes = (400, 2, 128, 2, 16)
        assert f(*sizes) > 0
        for i, size in enumerate(sizes):
            for wrong in (size + 2 ** 32, size - 2 ** 32, -1, 2 ** 31):
                refused(lambda: f(*sizes[:i], wrong, *sizes[i + 1:]))


def test_quantize_blocks_refused(lib):
    call = lib.redukt_op_quantize_blocks
    def args(**over):
        v = dict(dtype=0, rows=4, cols=100, block_rows=1, x=P, x_stride=100, codes=P, codes_stride=100, scales=P)
        v.update(over)
        return ctypes.byref(ops.QuantizeBlocks(**v))
    assert call(None, None) == BAD
    for over in (dict(dtype=3), dict(rows=1 << 31), dict(cols=1 << 31), dict(block_rows=0), dict(block_rows=64), dict(x=None), dict(codes=None),
                 dict(scales=None), dict(x=P + 1), dict(scales=P + 2), dict(x_stride=99), dict(codes_stride=99), dict(codes_stride=0),
                 dict(x_stride=-100), dict(rows=1 << 30, cols=1 << 20, x_stride=0, codes_stride=1 << 20), {}):
        assert call(args(**over), None) == BAD, over
    assert call(args(rows=0, x=None), None) == OK and call(args(cols=0, x=None, scales=None), None) == OK


def test_fp8_matmul_refused(lib):
    call = lib.redukt_op_fp8_matmul
    def args(**over):
        v = dict(dtype=0, m=4, n=6, k=100, x=P, x_stride=100, x_scales=P, w=P, w_stride=100, w_scales=P, bias=P, out=P, out_stride=6)
        v.update(over)
        return ctypes.byref(ops.Fp8Matmul(**v))
    assert call(None, None) == BAD
    for over in (dict(dtype=3), dict(m=1 << 31), dict(n=1 << 31), dict(k=(1 << 20) + 1), dict(x=None), dict(w=None), dict(x_scales=None),
                 dict(w_scales=None), dict(out=None), dict(x_scales=P + 2), dict(w_scales=P + 1), dict(bias=P + 2), dict(out=P + 1),
                 dict(out_stride=5), dict(x_stride=99), dict(w_stride=99), dict(x_stride=-100), {}):
        assert call(args(**over), None) == BAD, over
    assert call(args(m=0, out=None), None) == OK and call(args(n=0, out=None), None) == OK


def test_sample_refused(lib):
    call = lib.redukt_op_sample
    def args(**over):
        v = dict(dtype=0, rows=4, vocab=100, logits=P, logits_stride=100, u=P, temperature=1.0, top_p=1.0, min_p=0.0, top_k=0, temperatures=P,
                 top_ps=P, min_ps=P, top_ks=P, tokens=P)
        v.update(over)
        return ctypes.byref(ops.Sample(**v))
    assert call(None, None) == BAD
    for over in (dict(dtype=3), dict(rows=1 << 31), dict(vocab=0), dict(vocab=(1 << 20) + 1), dict(logits=None), dict(u=None), dict(tokens=None),
                 dict(logits=P + 1), dict(u=P + 2), dict(tokens=P + 2), dict(temperatures=P + 2), dict(top_ps=P + 1), dict(min_ps=P + 2),
                 dict(top_ks=P + 2), dict(logits_stride=99), dict(logits_stride=-100), {}):
        assert call(args(**over), None) == BAD, over
    assert call(args(rows=0, logits=None), None) == OK


# ---------------------------------------------------------------- the Python layer on its own

NEW = ("scan_step", "scan_chunk", "scan_grad", "quantize_blocks", "fp8_matmul", "sample")


class Recorded:
    """Stands for the library: what is called, with which arguments."""
    def __init__(self, lib):
        self.calls = []
        self.redukt_op_scan_chunk_workspace = lib.redukt_op_scan_chunk_workspace
        self.redukt_op_scan_grad_workspace = lib.redukt_op_scan_grad_workspace
        for name in NEW:
            setattr(self, "redukt_op_" + name, lambda *a: self.calls.append(a) or OK)


@pytest.fixture
def recorded(lib, monkeypatch):
    """The operators on CPU tensors, with nothing behind the checks of arguments."""
    r = Recorded(lib)
    monkeypatch.setattr(ops, "_device", lambda op, t: t.get_device() if isinstance(t, torch.Tensor) else ops._refuse(op))
    monkeypatch.setattr(ops, "_stream", lambda *a: None)
    monkeypatch.setattr(ops, "_load", lambda: r)
    return r


def refused(call):
    with pytest.raises(ffi.BackendError) as e:
        call()
    assert e.value.result == ffi.BackendResult.INVALID_ARGUMENT


def layer(T=3, ch=64, n=16, groups=1, dtype=BF16):
    z = lambda *s: torch.zeros(*s, dtype=dtype)  # noqa: E731
    return dict(x=z(T, ch), dt=z(T, ch), z=z(T, ch), b=z(T, groups, n), c=z(T, groups, n), a=torch.zeros(ch, n), d=torch.zeros(ch),
                dt_bias=torch.zeros(ch))


def calls():
    """Each operator on tensors of its own: (floating-point inputs and outputs by name, a call of them)."""
    cu = torch.tensor([0, 3], dtype=torch.int32)
    pool = lambda: torch.zeros(3, 64, 16)  # noqa: E731
    code = lambda r: torch.zeros(r, 128, dtype=E4M3)  # noqa: E731
    out = torch.zeros(3, 64, dtype=BF16)

    def grad(t):
        t = dict(t)
        grads = ops.ScanGrads(**{k[2:]: t.pop(k) for k in list(t) if k.startswith("g_")})
        return ops.scan_grad(cu_seqlens=cu, grads=grads, **t)

    g = {"g_" + k: v.clone() for k, v in layer().items()}
    return {"scan_step": (dict(layer(), states=pool(), out=out.clone()), lambda t: ops.scan_step(**t)),
            "scan_chunk": (dict(layer(), state_in=pool(), state_out=pool(), out=out.clone()), lambda t: ops.scan_chunk(cu_seqlens=cu, **t)),
            "scan_grad": (dict(layer(), dout=out.clone(), state_in=pool()[:1], dstate_out=pool()[:1], g_state_in=pool()[:1], **g), grad),
            "quantize_blocks": (dict(x=torch.zeros(3, 130), scales=torch.zeros(3, 2)), lambda t: ops.quantize_blocks(**t)),
            "fp8_matmul": (dict(x=code(3), x_scales=torch.ones(3, 1), w=code(5), w_scales=torch.ones(1, 1), bias=torch.zeros(5),
                                out=torch.zeros(3, 5)), lambda t: ops.fp8_matmul(**t)),
            "sample": (dict(logits=torch.zeros(3, 9), u=torch.zeros(3), temperature=torch.ones(3), top_p=torch.ones(3), min_p=torch.zeros(3)),
                       lambda t: ops.sample(**t))}


TENSORS = [(op, name) for op, (t, _) in calls().items() for name in t]


def test_the_calls_are_taken(recorded):
    for i, (tensors, call) in enumerate(calls().values()):
        call(tensors)
        assert len(recorded.calls) == i + 1


@pytest.mark.parametrize("op,name", TENSORS)
def test_every_tensor_that_asks_for_a_gradient_is_refused(recorded, op, name):
    tensors, call = calls()[op]
    tensors[name].requires_grad_()
    refused(lambda: call(tensors))
    assert not recorded.calls
    with torch.no_grad():
        call(tensors)
    assert len(recorded.calls) == 1


@pytest.mark.parametrize("op,name", [t for t in TENSORS if not (t[0] == "fp8_matmul" and t[1] in ("x", "w"))])
def test_every_tensor_with_a_tangent_is_refused(recorded, op, name):
    from torch.autograd import forward_ad

    tensors, call = calls()[op]
    with forward_ad.dual_level():
        call(tensors)
        refused(lambda: call(dict(tensors, **{name: forward_ad.make_dual(tensors[name], torch.ones_like(tensors[name]))})))
    assert len(recorded.calls) == 1


@pytest.mark.parametrize("op,name", TENSORS)
def test_what_is_no_tensor_or_of_another_type_is_refused(recorded, op, name):
    tensors, call = calls()[op]
    if not (op == "sample" and name in ("temperature", "top_p", "min_p")):
        refused(lambda: call(dict(tensors, **{name: 5})))
    refused(lambda: call(dict(tensors, **{name: tensors[name].to(torch.float64)})))
    refused(lambda: call(dict(tensors, **{name: tensors[name][None]})))
    refused(lambda: call(dict(tensors, **{name: "x"})))
    assert not recorded.calls


@pytest.mark.parametrize("op,written", [("scan_step", ["states", "out"]), ("scan_chunk", ["state_out", "out"]),
                                        ("scan_grad", ["g_x", "g_dt", "g_a", "g_b", "g_c", "g_d", "g_z", "g_dt_bias", "g_state_in"]),
                                        ("quantize_blocks", ["scales"]), ("fp8_matmul", ["out"])])
def test_what_a_call_writes_is_counted_as_written(recorded, op, written):
    tensors, call = calls()[op]
    before = {n: t._version for n, t in tensors.items()}
    call(tensors)
    for n, t in tensors.items():
        assert (t._version > before[n]) == (n in written), n


def test_outputs_of_no_floats_and_workspaces_are_counted_as_written(recorded):
    codes, tokens = torch.zeros(3, 16, dtype=E4M3), torch.zeros(3, dtype=torch.int32)
    ops.quantize_blocks(torch.zeros(3, 16), codes=codes)
    ops.sample(torch.zeros(3, 9), torch.zeros(3), out=tokens)
    cu = torch.tensor([0, 400], dtype=torch.int32)
    w1 = torch.zeros(ops.scan_chunk_workspace(400, 1, 64, 1, 16), dtype=torch.uint8)
    w2 = torch.zeros(ops.scan_grad_workspace(400, 1, 64, 1, 16), dtype=torch.uint8)
    ops.scan_chunk(cu_seqlens=cu, workspace=w1, **layer(400))
    ops.scan_grad(torch.zeros(400, 64, dtype=BF16), cu_seqlens=cu, workspace=w2, **layer(400))
    assert all(t._version == 1 for t in (codes, tokens, w1, w2))


def test_tensors_that_do_not_belong_together_are_refused(recorded):
    t = layer()
    pool = torch.zeros(3, 64, 16)
    for name, other in (("dt", torch.zeros(4, 64, dtype=BF16)), ("b", torch.zeros(3, 1, 8, dtype=BF16)), ("c", torch.zeros(3, 2, 16, dtype=BF16)),
                        ("a", torch.zeros(64, 8)), ("a", torch.zeros(16, 64).T), ("d", torch.zeros(65)), ("z", torch.zeros(3, 63, dtype=BF16)),
                        ("d", torch.zeros(128)[::2]), ("x", torch.zeros(64, 3, dtype=BF16).T)):
        refused(lambda: ops.scan_step(states=pool, **dict(t, **{name: other})))
    refused(lambda: ops.scan_step(states=torch.zeros(64, 3, 16).transpose(0, 1), **t))
    cu = torch.tensor([0, 3], dtype=torch.int32)
    refused(lambda: ops.scan_chunk(cu_seqlens=cu, state_in=pool, state_out=pool[:2], **t))
    refused(lambda: ops.scan_chunk(cu_seqlens=cu.long(), **t))
    refused(lambda: ops.scan_chunk(cu_seqlens=torch.zeros(0, dtype=torch.int32), **t))
    refused(lambda: ops.scan_grad(torch.zeros(3, 64, dtype=BF16), cu_seqlens=cu, state_in=pool, **t))
    refused(lambda: ops.scan_grad(torch.zeros(3, 64, dtype=BF16), cu_seqlens=cu, grads=(1, 2), **t))
    code, s = torch.zeros(3, 256, dtype=E4M3), torch.ones(3, 2)
    refused(lambda: ops.fp8_matmul(code, s[:, :1], code, s[:1]))
    refused(lambda: ops.fp8_matmul(code, s, code, s))
    refused(lambda: ops.fp8_matmul(code, torch.ones(2, 3).T, code, s[:1]))
    refused(lambda: ops.quantize_blocks(torch.zeros(3, 16), block_rows=2))
    refused(lambda: ops.sample(torch.zeros(3, 9), torch.zeros(3, 2)[:, 0]))
    refused(lambda: ops.sample(torch.zeros(3, 9), torch.zeros(3), top_k=torch.zeros(3)))
    assert not recorded.calls


def test_scan_refuses_tangents_and_states_of_other_sequences(recorded):
    from torch.autograd import forward_ad

    t, cu = layer(dtype=F32), torch.tensor([0, 3], dtype=torch.int32)
    refused(lambda: ops.scan(cu_seqlens=cu, state_in=torch.zeros(2, 64, 16), **t))
    with forward_ad.dual_level():
        refused(lambda: ops.scan(cu_seqlens=cu, **dict(t, x=forward_ad.make_dual(t["x"], torch.ones_like(t["x"])))))


BIG = 2 ** 32 + 5


def test_sizes_past_32_bits_are_refused(recorded):
    """They would arrive as what is left of them modulo 2^32.  (Tensors of stride 0: no memory is behind them.)"""
    t = {k: v[:1].expand(BIG, *v.shape[1:]) if k in ("x", "dt", "z", "b", "c") else v for k, v in layer(1).items()}
    refused(lambda: ops.scan_step(states=torch.zeros(1, 64, 16), out=t["x"], **t))
    refused(lambda: ops.scan_chunk(cu_seqlens=torch.zeros(2, dtype=torch.int32), out=t["x"], **t))
    one = torch.zeros(1, 1)
    byte = torch.zeros(1, 1, dtype=E4M3)
    refused(lambda: ops.quantize_blocks(one.expand(BIG, 1), codes=byte.expand(BIG, 1), scales=one.expand(BIG, 1)))
    refused(lambda: ops.fp8_matmul(byte.expand(1, BIG), one, byte.expand(1, BIG), one))
    refused(lambda: ops.sample(one.expand(1, BIG), torch.zeros(1)))
    assert not recorded.calls


def test_tensors_off_the_gpu_are_refused():
    for tensors, call in calls().values():
        refused(lambda: call(tensors))
    refused(lambda: ops.scan(cu_seqlens=torch.tensor([0, 3], dtype=torch.int32), **layer()))


# ---------------------------------------------------------------- the statements themselves

def test_the_gradients_statement_is_the_derivative():
    """scan_grad in 64 bits against autograd through scan in 64 bits."""
    g = torch.Generator().manual_seed(3)
    randn = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    T, ch, n, groups = 9, 6, 4, 2
    x = dict(x=randn(T, ch), dt=randn(T, ch), a=-torch.exp(randn(ch, n)), b=randn(T, groups, n), c=randn(T, groups, n), d=randn(ch), z=randn(T, ch),
             dt_bias=randn(ch))
    h0, dout, dlast = randn(ch, n), randn(T, ch), randn(ch, n)
    leaves = {k: v.clone().requires_grad_() for k, v in dict(x, h0=h0).items()}
    out, h = f64.scan(**leaves)
    ((out.v * dout).sum() + (h.v * dlast).sum()).backward()
    want = f64.scan_grad(dout, h0=h0, dfinal=dlast, **x)
    for k, v in leaves.items():
        assert torch.allclose(v.grad, want["state_in" if k == "h0" else k].v, rtol=1e-10, atol=1e-12), k


def test_the_bounds_hold_for_f32_and_notice_less():
    """The scan done in f32 is within its bound, and one with states of 16 bits is not."""
    g = torch.Generator().manual_seed(5)
    randn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    T, ch, n = 60, 5, 8
    x = dict(x=randn(T, ch), dt=randn(T, ch), a=-torch.exp(randn(ch, n)), b=randn(T, 1, n), c=randn(T, 1, n))
    out, _ = f64.scan(h0=torch.zeros(ch, n), **x)
    v, tol = f64.rounded(out, F32)

    def run(held):
        h, rows = torch.zeros(ch, n), []
        for t in range(T):
            s = torch.nn.functional.softplus(x["dt"][t])
            h = (torch.exp(s[:, None] * x["a"]) * h + (s * x["x"][t])[:, None] * x["b"][t]).to(held).float()
            rows.append((h * x["c"][t]).sum(-1))
        return torch.stack(rows).double()

    assert ((run(F32) - v).abs() <= tol).all() and not ((run(BF16) - v).abs() <= tol).all()


def test_e4m3_values_are_torchs():
    every = torch.arange(256, dtype=torch.uint8).view(E4M3).float()
    every = every[~every.isnan()]
    mids = torch.cat([(every[:-1] + every[1:]) / 2, every, every * 1.01])
    mids = mids[mids.abs() <= 448]
    assert np.array_equal(f64.to_e4m3(mids.double().numpy()), mids.to(E4M3).double().numpy())


def test_drawing_by_hand():
    l = [1.0, 3.0, 2.0, 3.0, float("-inf"), float("nan")]
    e = np.exp(-1.0), np.exp(-2.0)
    total = 2 + e[0] + e[1]
    assert f64.draw(l, 0.0) == 0 and f64.draw(l, (e[1] + 0.5) / total) == 1 and f64.draw(l, (e[1] + 1.01) / total) == 2
    assert f64.draw(l, 0.999) == 3 and f64.draw(l, 0.3, top_k=1) == 1 and f64.draw(l, 0.6, top_k=2) == 3
    assert f64.draw(l, 0.3, temperature=0.0) == 1 and f64.draw([float("-inf")] * 3, 0.5) == -1
    assert f64.draw(l, 0.99, top_p=0.3) == 1 and f64.draw(l, 0.99, min_p=0.5) == 3


def test_settings_that_are_no_numbers_are_refused(recorded):
    for over in (dict(top_k=float("inf")), dict(top_k=float("nan")), dict(temperature=10 ** 400), dict(top_p="half"), dict(min_p=[0.1])):
        refused(lambda: ops.sample(torch.zeros(3, 9), torch.zeros(3), out=torch.zeros(3, dtype=torch.int32), **over))
    assert not recorded.calls
